"""Operators of a serving step around a paged key-value cache: what is measured of them.

Three operators.  Queries, keys and values are Q8.8 (int16), logits Q16.16 (int32).

* ``append``: rows [q | k | v] of many requests.  Row r of request b, one of its n_b
  rows offsets[b] .. offsets[b+1]-1, is at position lengths[b] - n_b + r - offsets[b].
  Queries and keys are rotated by the table's row of that position,

      x0' = sat16(rnd8(x0 c - x1 s)),  x1' = sat16(rnd8(x1 c + x0 s))    pairs (i, i + d/2)

  keys and values go to their place in the pages that the request's table row names.

* ``attend``: a block of 1 to 8 rows per request over the pages, row j of n_b seeing the
  first lengths[b] - n_b + j + 1 positions (none: zeros).  64 positions at a time, in order:

      s    = score, per product rounded to Q16.16 in four saturating banks, times fm(1/sqrt(d))
      m    = running maximum,  P = exp(s - m) cut off to Q2.14,  f = exp(m_before - m) likewise
      sum  = sat32(rnd16(sum 4f) + sum of 4P)
      tv   = sat16(rnd8(rnd6(sum of rnd4(P sat16(16 v)))))
      acc  = sat32(sat32(rnd16(acc 4f)) + 256 tv)
      out  = sat16(rnd24(acc 256 sat16(rnd8(2^32 / max(sum, 16)))))

* ``logprob``: of rows of logits z at temperature T, with d_v = (max z - z_v) / (2^16 T):
  the log probability and the rank of a given token, the entropy in nats, and the most
  likely tokens with theirs.  INT32_MIN excludes a token, T <= 1e-6 leaves the first maximum.

Results of the first two are whole numbers that both forms reach exactly; those of the
third are 32-bit floats, ranks and tokens whole numbers (ties to the lowest index).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
NONE = -(2**31)  # a logit that excludes its token
NO_TOKEN = -1  # 0xffffffff
UNTOUCHED = 7777  # what rows behind the last request hold before and after


def _framework():
    folder = os.path.join(os.getcwd(), "llm-accel_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import llmx

    return llmx


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    qwen = {"heads": 16, "kv": 2, "dim": 128}
    return [
        # a decode step of 64 requests, each row to its own place
        {"name": "append_64req", "op": "append", **qwen, "page": 16, "requests": 64, "block": 1, "length": 2048, "pad": 0},
        # four prompts, one piece of 2048 tokens each
        {"name": "append_prompts", "op": "append", **qwen, "page": 64, "requests": 4, "block": 2048, "length": 4096, "pad": 5},
        # one new token of one request: latency counts
        {"name": "attend_1req_513", "op": "attend", **qwen, "page": 16, "requests": 1, "block": 1, "length": 513, "even": True, "pad": 0},
        # blocks of the last token and four drafts, to be verified
        {"name": "attend_drafts", "op": "attend", **qwen, "page": 32, "requests": 8, "block": 5, "length": 1100, "even": False, "pad": 0},
        # sizes that fit no tile: five query heads to a key head, pages that end inside a tile
        {"name": "attend_odd", "op": "attend", "heads": 10, "kv": 2, "dim": 80, "page": 24, "requests": 13, "block": 3,
         "length": 777, "even": False, "pad": 3},
        # one request with a long text
        {"name": "attend_1req_32k", "op": "attend", **qwen, "page": 64, "requests": 1, "block": 1, "length": 32768, "even": True, "pad": 0},
        # a decode step of 64 requests of every length
        {"name": "attend_64req", "op": "attend", **qwen, "page": 16, "requests": 64, "block": 1, "length": 2304, "even": False, "pad": 1},
        # the same with long texts
        {"name": "attend_64req_8k", "op": "attend", **qwen, "page": 64, "requests": 64, "block": 1, "length": 8192, "even": True, "pad": 0},
        # one sampled token and five alternatives
        {"name": "logprob_1row", "op": "logprob", "rows": 1, "vocab": 151936, "top": 5, "ragged": False},
        # a small vocabulary, some tokens excluded
        {"name": "logprob_odd", "op": "logprob", "rows": 77, "vocab": 32003, "top": 7, "ragged": True},
        # a decode step of 64 requests, all the alternatives that an interface offers
        {"name": "logprob_64rows", "op": "logprob", "rows": 64, "vocab": 151936, "top": 20, "ragged": False},
        # a prompt's tokens scored
        {"name": "logprob_prompt", "op": "logprob", "rows": 512, "vocab": 151936, "top": 1, "ragged": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    if rng.random() < 0.5:
        return {"heads": 16, "kv": 2, "dim": 128}
    kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    return {"heads": kv * group, "kv": kv, "dim": rng.choice([16, 32, 48, 64, 80, 96, 112, 128])}


def draw(rng):
    kind = rng.random()
    if kind < 0.25:
        s = _heads(rng)
        requests = _log(rng, 1, 128)
        block = _log(rng, 1, max(1, 8192 * 2560 // ((s["heads"] + 2 * s["kv"]) * s["dim"]) // requests))
        block = min(block, 4096)
        return {"op": "append", **s, "page": rng.choice([8, 16, 24, 32, 64, 256]), "requests": requests, "block": block,
                "length": min(block + _log(rng, 1, 4096), 2**17 // requests + block), "pad": rng.randint(0, 3)}
    if kind < 0.7:
        s = _heads(rng)
        requests, block = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 3, 5, 8])
        most = 64 * 8192 * 16 * 128 // (requests * block * s["heads"] * s["dim"])
        return {"op": "attend", **s, "page": rng.choice([8, 16, 24, 32, 64, 256]), "requests": requests, "block": block,
                "length": _log(rng, 1, min(most, 32768, 2**19 // requests)), "even": rng.random() < 0.3, "pad": rng.randint(0, 3)}
    return {"op": "logprob", "rows": _log(rng, 1, 512), "vocab": _log(rng, 40, 151936), "top": rng.choice([0, 1, 5, 20, 32]),
            "ragged": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# plans that follow from a case alone
# ---------------------------------------------------------------------------
def _plan(case):
    """(rows, length) of each request: the case's, or spread down to an empty one."""
    n, block, length = case["requests"], case["block"], case["length"]
    if case["op"] == "append":  # lengths include the rows that are appended
        return [(block - b * 3 % (block // 2 + 1), length - (b * 37) % (length - block + 1)) for b in range(n)]
    if case["even"]:
        return [(block, length)] * n
    out = []
    for b in range(n):
        rows = block - b % min(block, 3)
        out.append((rows, 0 if b % 11 == 10 else max(rows, length * (n - b) // n)))
    return out


def _counts(case):
    """Rows of all requests, rows of the arrays."""
    total = sum(r for r, _ in _plan(case))
    return total, total + case["pad"]


def _score_scale(dim):
    return math.floor(256 / math.sqrt(dim) + 0.5) * 256


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (_prepare_logprob if case["op"] == "logprob" else _prepare_paged)(case, g)


def _whole(g, shape, sigma):
    return torch.randn(shape, generator=g, device=DEV).mul_(sigma).round_().clamp_(-32768, 32767).to(torch.int16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_paged(case, g):
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    plan, (total, rows) = _plan(case), _counts(case)
    need = [-(-length // page) for _, length in plan]
    pages = sum(need) + 2
    # the pages lie in any order; places of a table that no position uses name no page
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    width = max(need) + 1
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    offsets = [0]
    for r, _ in plan:
        offsets.append(offsets[-1] + r)
    s = {"op": case["op"], "heads": heads, "kv": kv, "dim": dim, "page": page, "plan": plan, "rows": rows, "total": total,
         "offsets": _i32(offsets), "lengths": _i32([length for _, length in plan]), "table": table, "pages": pages}
    shape = (pages, kv, page, dim)
    if case["op"] == "append":
        x = _whole(g, (rows, (heads + 2 * kv) * dim), 400)
        positions = max(length for _, length in plan)
        # angles of far positions need 64 bits
        i = torch.arange(dim // 2, dtype=torch.float64, device=DEV)
        angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * (1e6 ** (-2 * i / dim))
        rope = torch.cat([angle.cos(), angle.sin()], 1).mul_(256).round_().to(torch.int16)
        s.update(x=x, rope=rope, k=torch.zeros(shape, dtype=torch.int16, device=DEV), v=torch.zeros(shape, dtype=torch.int16, device=DEV),
                 q=torch.full((rows, heads * dim), UNTOUCHED, dtype=torch.int16, device=DEV))
    else:
        # some channels of the keys are large, a few values beyond the +-8 of a Q4.12 operand
        wide = (torch.rand((dim,), generator=g, device=DEV) < 0.06).float().mul_(4).add_(1)
        k = torch.randn(shape, generator=g, device=DEV).mul_(300).mul_(wide).round_().clamp_(-32768, 32767).to(torch.int16)
        s.update(q=_whole(g, (rows, heads * dim), 330), k=k, v=_whole(g, shape, 256),
                 out=torch.full((rows, heads * dim), UNTOUCHED, dtype=torch.int16, device=DEV))
    if own:
        llmx = _framework()
        longest = max(max(length for _, length in plan), 1)
        block = min(max(r for r, _ in plan), 8)
        s.update(llmx=llmx, longest=longest, plan_handle=llmx.Paged(heads, kv, dim, page, case["requests"], block, longest,
                                                                      max(sum(length for _, length in plan), 1),
                                                                      stream=torch.cuda.current_stream().cuda_stream))
    return s


def _prepare_logprob(case, g):
    rows, vocab = case["rows"], case["vocab"]
    z = torch.randn((rows, vocab), generator=g, device=DEV) * 2.5
    likely = torch.randint(0, vocab, (rows, 12), generator=g, device=DEV)
    z.scatter_add_(1, likely, torch.rand((rows, 12), generator=g, device=DEV) * 14)
    # the given tokens: one of the likely ones mostly, any one in four
    tokens = torch.where(torch.rand((rows,), generator=g, device=DEV) < 0.75, likely[:, 0],
                         torch.randint(0, vocab, (rows,), generator=g, device=DEV)).to(torch.int32)
    logits = (z * 65536).round_().clamp_(-(2.0**31) + 256, 2.0**31 - 256).to(torch.int32)
    del z
    temperature = torch.ones((rows,), device=DEV)
    if case["ragged"]:
        logits.masked_fill_(torch.rand((rows, vocab), generator=g, device=DEV) < 0.25, NONE)
        temperature = torch.rand((rows,), generator=g, device=DEV) + 0.5
        temperature[3::7] = 0.0  # greedy rows among the others
    s = {"op": "logprob", "logits": logits, "tokens": tokens, "temperature": temperature, "top": case["top"]}
    if own:
        llmx = _framework()
        new = lambda shape, kind: torch.empty(shape, dtype=kind, device=DEV)  # noqa: E731
        s.update(llmx=llmx, work=new((max(llmx.logprobs_workspace_bytes(rows, vocab, case["top"]), 1),), torch.uint8),
                 logprob=new((rows,), torch.float32), rank=new((rows,), torch.int32), entropy=new((rows,), torch.float32),
                 top_tokens=new((rows, case["top"]), torch.int32), top_logprobs=new((rows, case["top"]), torch.float32))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return _RUN[s["op"], own](s)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_append(s):
    s["plan_handle"].append(s["x"].data_ptr(), s["rows"], s["offsets"].data_ptr(), s["lengths"].data_ptr(), len(s["plan"]),
                            s["rope"].data_ptr(), s["rope"].shape[0], s["table"].data_ptr(), s["table"].shape[1], s["k"].data_ptr(),
                            s["v"].data_ptr(), s["pages"], s["q"].data_ptr(), stream=_stream())
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attend(s):
    s["plan_handle"].attention(s["q"].data_ptr(), s["rows"], s["offsets"].data_ptr(), s["lengths"].data_ptr(), len(s["plan"]),
                               s["table"].data_ptr(), s["table"].shape[1], s["k"].data_ptr(), s["v"].data_ptr(), s["pages"],
                               s["out"].data_ptr(), longest=s["longest"], stream=_stream())
    return s["out"]


def _own_logprob(s):
    top = s["top"]
    s["llmx"].token_logprobs(s["logits"].data_ptr(), s["logits"].shape[0], s["logits"].shape[1], s["tokens"].data_ptr(),
                             s["temperature"].data_ptr(), top, s["logprob"].data_ptr(), s["rank"].data_ptr(), s["entropy"].data_ptr(),
                             s["top_tokens"].data_ptr() if top else None, s["top_logprobs"].data_ptr() if top else None,
                             s["work"].data_ptr(), s["work"].numel(), stream=_stream())
    return {f: s[f] for f in ("logprob", "rank", "entropy", "top_tokens", "top_logprobs")}


def _rnd(v, k):
    return (v + (1 << (k - 1))) >> k


def _sat16(v):
    return v.clamp(-32768, 32767)


def _sat32(v):
    return v.clamp(-(2**31), 2**31 - 1)


def _plain_append(s):
    heads, kv, dim, page, total = s["heads"], s["kv"], s["dim"], s["page"], s["total"]
    counts = (s["offsets"][1:] - s["offsets"][:-1]).long()
    owner = torch.repeat_interleave(torch.arange(len(s["plan"]), device=DEV), counts, output_size=total)
    position = s["lengths"].long()[owner] - counts[owner] + torch.arange(total, device=DEV) - s["offsets"].long()[owner]
    x = s["x"][:total].view(total, heads + 2 * kv, dim)
    turn = s["rope"][position].int()[:, None]
    c, sn = turn[..., :dim // 2], turn[..., dim // 2:]
    x0, x1 = x[:, :heads + kv, :dim // 2].int(), x[:, :heads + kv, dim // 2:].int()
    rotated = torch.cat([_sat16(_rnd(x0 * c - x1 * sn, 8)), _sat16(_rnd(x1 * c + x0 * sn, 8))], 2).to(torch.int16)
    where = s["table"].long()[owner, position // page], position % page
    s["q"][:total] = rotated[:, :heads].reshape(total, heads * dim)
    s["k"][where[0], :, where[1]] = rotated[:, heads:]
    s["v"][where[0], :, where[1]] = x[:, heads + kv:]
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _exp_table():
    """exp(x / 256) of x = -2048 .. 0, cut off to Q2.14."""
    x = torch.arange(-2048, 1, dtype=torch.float64, device=DEV)
    return torch.floor(torch.exp(x / 256) * 16384).int()


def _plain_attend(s):
    heads, kv, dim, page = s["heads"], s["kv"], s["dim"], s["page"]
    group, at = heads // kv, 0
    exps = _exp_table()
    out = torch.full_like(s["out"], UNTOUCHED)
    for b, (rows, length) in enumerate(s["plan"]):
        q = s["q"][at:at + rows].view(rows, kv, group, dim)
        if length == 0:
            out[at:at + rows] = 0
            at += rows
            continue
        position = torch.arange(length, device=DEV)
        where = s["table"][b].long()[position // page], position % page
        k, v = s["k"][where[0], :, where[1]], s["v"][where[0], :, where[1]]  # [length][kv][dim]
        seen = length - rows + 1 + torch.arange(rows, device=DEV)
        res = [_plain_head(q[:, h].reshape(rows * group, dim), k[:, h], v[:, h], seen.repeat_interleave(group), exps) for h in range(kv)]
        out[at:at + rows] = torch.stack([r.view(rows, group * dim) for r in res], 1).reshape(rows, heads * dim)
        at += rows
    return out


def _plain_head(q, k, v, seen, exps):
    """Queries q [n][dim] against one key head's k and v [length][dim]."""
    n, dim = q.shape
    length = k.shape[0]
    tiles = -(-length // 64)
    wk, wv = _sat16(k.int() * 16), _sat16(v.int() * 16)
    piece = max(1, 2**26 // (n * dim))  # positions whose products are formed at once
    score = []
    for a in range(0, length, piece):
        products = _rnd(q.int()[:, None] * wk[None, a:a + piece], 4)
        banks = _sat32(products.view(n, -1, dim // 4, 4).sum(2, dtype=torch.int64))  # 31 products of a bank never saturate
        total = _sat32(_rnd(_sat32(banks.sum(2)) * _score_scale(dim), 16))
        score.append(_sat16(_rnd(total, 8)).int())
    score = torch.cat(score, 1)
    pad = tiles * 64 - length
    live = torch.arange(tiles * 64, device=DEV)[None] < seen[:, None]
    score = torch.nn.functional.pad(score, (0, pad), value=-32768).masked_fill(~live, -32768).view(n, tiles, 64)
    live = live.view(n, tiles, 64)
    top = score.amax(2).cummax(1).values
    before = torch.nn.functional.pad(top[:, :-1], (1, 0), value=-32768)
    index = lambda d: _sat16(d).clamp(-2048, 0).long() + 2048  # noqa: E731
    p = exps[index(score - top[:, :, None])] * live
    factor = exps[index(before - top)].long() * 4
    sums = p.sum(2, dtype=torch.int64) * 4
    wv = torch.nn.functional.pad(wv, (0, 0, 0, pad)).view(tiles, 64, dim)
    piece = max(1, 2**20 // (n * dim))  # tiles at once
    tv = []
    for a in range(0, tiles, piece):
        products = _rnd(p[:, a:a + piece, :, None] * wv[None, a:a + piece], 4)
        tv.append(_sat16(_rnd(_rnd(_sat32(products.sum(2, dtype=torch.int64)), 6), 8)) * 256)
    tv = torch.cat(tv, 1)
    norm = torch.zeros((n,), dtype=torch.int64, device=DEV)
    acc = torch.zeros((n, dim), dtype=torch.int64, device=DEV)
    for t in range(tiles):
        f = factor[:, t]
        norm = _sat32(_rnd(norm * f, 16) + sums[:, t])
        acc = _sat32(_sat32(_rnd(acc * f[:, None], 16)) + tv[:, t])
    inverse = _sat16(_rnd((1 << 32) // norm.clamp_min(16), 8))
    return _sat16(_rnd(acc * (inverse * 256)[:, None], 24)).to(torch.int16)


def _plain_logprob(s):
    z, tokens, top = s["logits"].long(), s["tokens"].long(), s["top"]
    rows, vocab = z.shape
    live = z != NONE
    most = z.amax(1, keepdim=True)
    greedy = ~(s["temperature"] > 1e-6)[:, None]
    # sums of a whole vocabulary and logarithms next to 0: in 64 bits
    t = torch.where(greedy[:, 0], 1.0, s["temperature"].double())[:, None] * 65536
    d = (most - z).double() / t
    place = torch.arange(vocab, device=DEV)
    first = torch.where(z == most, place, vocab).amin(1, keepdim=True)
    w = torch.exp(-d).masked_fill_(~live | (place == first), 0)  # of all but the first maximum
    w.masked_fill_(greedy, 0)
    rest = w.sum(1)
    log_sum = torch.log1p(rest)
    entropy = log_sum + (w * d).sum(1) / (1 + rest)
    entropy.masked_fill_(~live.any(1), 0)

    def of(ids):  # [rows][n]
        lp = -d.gather(1, ids) - log_sum[:, None]
        return torch.where(live.gather(1, ids) & (~greedy | (ids == first)), lp, -math.inf)

    at = tokens[:, None]
    mine = z.gather(1, at)
    rank = ((z > mine) | ((z == mine) & (place < at))).sum(1)
    rank = torch.where(live.gather(1, at)[:, 0], rank, -1)
    # one number per token that orders by logit, then by index
    best = (z * 2**22 - place).topk(top, 1).values
    ids = (-best) & (2**22 - 1)
    known = live.gather(1, ids)
    return {"logprob": of(at)[:, 0].float(), "rank": rank.int(), "entropy": entropy.float(),
            "top_tokens": torch.where(known, ids, NO_TOKEN).int(), "top_logprobs": of(ids).float()}


_RUN = {("append", False): _plain_append, ("attend", False): _plain_attend, ("logprob", False): _plain_logprob,
        ("append", True): _own_append, ("attend", True): _own_attend, ("logprob", True): _own_logprob}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "logprob":
        n = case["rows"] * case["vocab"]
        # per logit: a difference, its scaling, an exponential, two sums, three comparisons
        return {"bytes": 4 * n + case["rows"] * (20 + 8 * case["top"]), "flops": 8 * n}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    plan, (total, _) = _plan(case), _counts(case)
    if case["op"] == "append":
        positions = sum(min(r, length) for r, length in plan)
        # six operations to a rotated pair; the table's rows, read once each
        return {"bytes": 2 * total * dim * 2 * (heads + 2 * kv) + 2 * dim * min(positions, max(length for _, length in plan)),
                "flops": 3 * total * (heads + kv) * dim}
    pairs = sum(max(0, length - r + 1 + j) for r, length in plan for j in range(r))
    return {"bytes": 4 * kv * dim * sum(length for _, length in plan) + 4 * total * heads * dim, "flops": 4 * heads * dim * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, on the host
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "logprob" and case["rows"] * case["vocab"] > 1e8:
        return None
    if case["op"] == "append" and _counts(case)[0] * (case["heads"] + 2 * case["kv"]) * case["dim"] > 3e7:
        return None
    if case["op"] == "attend":
        tiles = sum(r * -(-length // 64) for r, length in _plan(case))
        if tiles > 3000 or tiles * 64 * case["heads"] * case["dim"] > 1.5e8:
            return None
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    h = {f: (v.cpu().numpy() if isinstance(v, torch.Tensor) else v) for f, v in s.items()}
    return {"append": _exact_append, "attend": _exact_attend, "logprob": _exact_logprob}[case["op"]](h)


def _rows_of(h):
    """(row, request, position) of every row of a request."""
    for b, length in enumerate(h["lengths"].tolist()):
        first, end = int(h["offsets"][b]), int(h["offsets"][b + 1])
        for r in range(first, end):
            yield r, b, length - (end - r)


def _exact_append(h):
    heads, kv, dim, page = h["heads"], h["kv"], h["dim"], h["page"]
    half = dim // 2
    q, k, v = h["q"].copy(), h["k"].copy(), h["v"].copy()
    for r, b, position in _rows_of(h):
        x = h["x"][r].astype(np.int64).reshape(heads + 2 * kv, dim)
        c, sn = h["rope"][position, :half].astype(np.int64), h["rope"][position, half:].astype(np.int64)
        y = x.copy()
        y[:heads + kv, :half] = x[:heads + kv, :half] * c - x[:heads + kv, half:] * sn
        y[:heads + kv, half:] = x[:heads + kv, half:] * c + x[:heads + kv, :half] * sn
        y[:heads + kv] = np.clip(np.floor_divide(y[:heads + kv] + 128, 256), -32768, 32767)
        q[r] = y[:heads].reshape(-1)
        p = int(h["table"][b, position // page])
        k[p, :, position % page] = y[heads:heads + kv]
        v[p, :, position % page] = y[heads + kv:]
    return {"q": q, "k": k, "v": v}


def _exact_attend(h):
    heads, kv, dim, page = h["heads"], h["kv"], h["dim"], h["page"]
    lo, hi = -(2**31), 2**31 - 1
    # the exponentials, cut off: floor(exp(-i / 256) 2^14)
    exps = np.array([math.floor(math.exp(-i / 256) * 16384) for i in range(2049)], np.int64)
    scale = math.floor(256 / math.sqrt(dim) + 0.5) * 256
    out = np.full((h["rows"], heads * dim), UNTOUCHED, np.int16)
    for b, length in enumerate(h["lengths"].tolist()):
        first, end = int(h["offsets"][b]), int(h["offsets"][b + 1])
        where = [(int(h["table"][b, p // page]), p % page) for p in range(length)]
        cache = [np.stack([a[i, :, j] for i, j in where]).astype(np.int64) if where else None for a in (h["k"], h["v"])]
        for r in range(first, end):
            seen = length - (end - r) + 1
            q = h["q"][r].astype(np.int64).reshape(heads, dim)
            best, norm, acc = np.full(heads, -32768), np.zeros(heads, np.int64), np.zeros((heads, dim), np.int64)
            for t in range(0, max(seen, 0), 64):
                k, v = (np.clip(a[t:min(t + 64, seen)] * 16, -32768, 32767).repeat(heads // kv, 1) for a in cache)  # [positions][heads][dim]
                banks = np.zeros((4, len(k), heads), np.int64)
                for e in range(dim):
                    banks[e % 4] = np.clip(banks[e % 4] + ((q[:, e] * k[:, :, e] + 8) >> 4), lo, hi)
                score = np.clip(banks.sum(0), lo, hi)
                score = np.clip((((score * scale + 32768) >> 16) + 128) >> 8, -32768, 32767)  # [positions][heads]
                now = np.maximum(best, score.max(0))
                f = 4 * exps[np.minimum(now - best, 2048)]
                p = exps[np.minimum(now - score, 2048)]
                best = now
                norm = np.clip(((norm * f + 32768) >> 16) + 4 * p.sum(0), lo, hi)
                acc = np.clip((acc * f[:, None] + 32768) >> 16, lo, hi)
                banks = np.zeros((4, heads, dim), np.int64)
                for j in range(len(v)):
                    banks[j % 4] = np.clip(banks[j % 4] + ((p[j][:, None] * v[j] + 8) >> 4), lo, hi)
                tv = (np.clip(banks.sum(0), lo, hi) * 1024 + 32768) >> 16
                acc = np.clip(acc + 256 * np.clip((tv + 128) >> 8, -32768, 32767), lo, hi)
            inverse = np.clip(((1 << 32) // np.maximum(norm, 16) + 128) >> 8, -32768, 32767)
            out[r] = np.clip((acc * (inverse * 256)[:, None] + (1 << 23)) >> 24, -32768, 32767).reshape(-1)
    return out


def _exact_logprob(h):
    rows, vocab = h["logits"].shape
    top = h["top"]
    logprob, entropy = np.full(rows, -np.inf), np.zeros(rows)
    rank = np.full(rows, -1, np.int32)
    ids, lps = np.full((rows, top), NO_TOKEN, np.int32), np.full((rows, top), -np.inf)
    for r in range(rows):
        z = h["logits"][r].astype(np.int64)
        live = np.nonzero(z != NONE)[0]
        if len(live) == 0:
            continue
        z = z[live]
        first = int(np.argmax(z))
        t = float(h["temperature"][r])
        if t > 1e-6:
            d = (z[first] - z) / (65536.0 * t)
        else:
            d = np.where(np.arange(len(z)) == first, 0.0, np.inf)
        w = np.exp(-d)
        w[first] = 0
        rest = w.sum()
        log_sum = math.log1p(rest)
        entropy[r] = log_sum + (w[w > 0] * d[w > 0]).sum() / (1 + rest)
        lp = -d - log_sum
        n = min(top, len(z))
        if n:
            near = np.nonzero(z >= np.partition(z, len(z) - n)[len(z) - n])[0]
            near = near[np.argsort(-z[near], kind="stable")][:n]
            ids[r, :n], lps[r, :n] = live[near], lp[near]
        at = int(np.searchsorted(live, h["tokens"][r]))
        if at < len(z) and live[at] == h["tokens"][r]:
            rank[r], logprob[r] = (z > z[at]).sum() + (z[:at] == z[at]).sum(), lp[at]
    return {"logprob": logprob, "rank": rank, "entropy": entropy, "top_tokens": ids, "top_logprobs": lps}
