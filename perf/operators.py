"""The operators that serve several requests at once: what is measured of them.

Two operators, used one after the other in a speculative serving step.

* ``project``: a projection that every request shares, with each row's own
  low-rank adapter beside it.  Rows x are Q8.8, weights W, adapter matrices A
  (down) and B (up) and the adapter's scale s are Q4.12, all int16:

      t[i][j] = sat16(rnd24(s[a] * sum_k A[a][j][k] x[i][k]))          Q8.8
      y[i][n] = sum_k W[n][k] x[i][k] + sum_j B[a][n][j] t[i][j]        exact
      out     = sat32(rnd4(y))  Q16.16, or sat16(rnd8(sat32(rnd4(y))))  Q8.8

  with a = slot[i] (none for -1) and rndk(v) = floor(v / 2^k + 1/2).

* ``verify``: rejection sampling of drafted tokens from given random numbers.
  Rows of Q16.16 logits become whole-number weights (weight()), their sums are
  exact, and p and q are Q0.40:

      P[v] = (w[v] * floor(2^62 / (S >> h))) >> (22 + h)   S = sum w, S >> h in [2^31, 2^32)
      draft j is accepted while  U[j] * Q[x_j] < 2^32 * P[x_j]
      then one token of max(0, P - Q) at the first rejected row (of P if that is
      all zero), or of P at the last row: the first v whose running sum exceeds
      floor(V * total / 2^32).

Every result is a whole number that both forms have to reach exactly, so the
plain form forms its long dot products in 64-bit floats, where they are whole
numbers below 2^53: 32-bit floats hold only 24 bits of a 42-bit sum.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
NONE = -(2**31)  # a logit that excludes its token
# 2^x = 1 + x (C0 + x (C1 + ...)) on [-1/2, 1/2], each step rounded to 32 bits
COEF = (0.6931470036506653, 0.24022242426872253, 0.05550733581185341, 0.009671512991189957, 0.001326472614891827)
LOG2E_16 = float.fromhex("0x1.715476p-16")  # log2(e) / 2^16, of Q16.16 differences


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
    return [
        # one decoded token of one request through Q/K/V with its adapter: latency counts
        {"name": "qkv_1row", "op": "project", "rows": 1, "per": 1, "k": 2048, "n": 2560, "slots": 4, "rank": 16, "wide": False},
        # a prompt block of one request through Down
        {"name": "down_8rows", "op": "project", "rows": 8, "per": 8, "k": 11008, "n": 2048, "slots": 4, "rank": 16, "wide": False},
        # a decode step of 16 requests through Gate/Up, each with an adapter of its own
        {"name": "gate_up_16req", "op": "project", "rows": 16, "per": 1, "k": 2048, "n": 22016, "slots": 16, "rank": 32, "wide": False},
        # 8 requests' blocks of 5 rows (4 drafts and the last token) through the LM head: logits to verify
        {"name": "lm_head_40rows", "op": "project", "rows": 40, "per": 5, "k": 2048, "n": 151936, "slots": 8, "rank": 8, "wide": True},
        # sizes that fit no tile, ranks and requests ragged
        {"name": "odd_77rows", "op": "project", "rows": 77, "per": 3, "k": 1096, "n": 4999, "slots": 20, "rank": 13, "wide": True},
        # 64 requests' blocks of 8 rows through Gate, four adapters among them
        {"name": "gate_512rows", "op": "project", "rows": 512, "per": 8, "k": 2048, "n": 11008, "slots": 4, "rank": 64, "wide": False},
        # one request whose drafts were copied from its prompt: no draft distribution
        {"name": "copied_4drafts", "op": "verify", "requests": 1, "drafts": 4, "vocab": 151936, "model": False, "ragged": False},
        # one request, a full block of drafts from a draft model
        {"name": "one_7drafts", "op": "verify", "requests": 1, "drafts": 7, "vocab": 151936, "model": True, "ragged": False},
        # a small vocabulary, some tokens excluded, requests with fewer drafts or none
        {"name": "small_vocab_ragged", "op": "verify", "requests": 5, "drafts": 3, "vocab": 997, "model": True, "ragged": True},
        # sampling alone: no drafts
        {"name": "sample_64", "op": "verify", "requests": 64, "drafts": 0, "vocab": 151936, "model": False, "ragged": False},
        # a serving batch
        {"name": "batch32_ragged", "op": "verify", "requests": 32, "drafts": 4, "vocab": 151936, "model": True, "ragged": True},
        # the largest batch, full blocks
        {"name": "batch64_7drafts", "op": "verify", "requests": 64, "drafts": 7, "vocab": 151936, "model": True, "ragged": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        k = max(64, _log(rng, 64, 11008) // 8 * 8)
        n = min(_log(rng, 64, 151936), 151936 * 2048 // k)
        rows = _log(rng, 1, 512)
        rows = max(1, min(rows, 64 * 151936 * 2048 // (2 * n * k)))
        per = min(rows, rng.choice([1, 1, 2, 3, 5, 8]))
        return {"op": "project", "rows": rows, "per": per, "k": k, "n": n, "slots": _log(rng, 1, 48),
                "rank": _log(rng, 1, 128 if rows <= 64 else 64), "wide": rng.random() < 0.5}
    requests, drafts = _log(rng, 1, 64), rng.randint(0, 7)
    model = drafts > 0 and rng.random() < 0.7
    return {"op": "verify", "requests": requests, "drafts": drafts, "vocab": _log(rng, 32, 151936), "model": model,
            "ragged": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# plans that follow from a case alone
# ---------------------------------------------------------------------------
def _ranks(case):
    """Rank of each slot: the case's, three quarters and a half of it in turn."""
    r = case["rank"]
    return [max(1, (r * (4 - s % 3) + 3) // 4) for s in range(case["slots"])]


def _slots_of_requests(case):
    """Requests take the slots in turn; one in nine has no adapter."""
    requests = -(-case["rows"] // case["per"])
    return [-1 if q % 9 == 8 else q % case["slots"] for q in range(requests)]


def _counts(case):
    """Drafts of each request."""
    b, k = case["requests"], case["drafts"]
    return [k - (q * 3 % (k + 1) if case["ragged"] else 0) for q in range(b)]


def _whole(g, shape, sigma, top=32767):
    return (torch.randn(shape, generator=g, device=DEV) * sigma).round_().clamp_(-top - 1, top).to(torch.int16)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (_prepare_project if case["op"] == "project" else _prepare_verify)(case, g)


def _prepare_project(case, g):
    rows, k, n, slots, rank = (case[f] for f in ("rows", "k", "n", "slots", "rank"))
    ranks = _ranks(case)
    x = torch.randn((rows, k), generator=g, device=DEV) * 256
    # a few channels of every row are far larger than the rest
    big = torch.rand((k,), generator=g, device=DEV) < 0.004
    x = torch.where(big, x * 30, x).round_().clamp_(-32768, 32767).to(torch.int16)
    w = _whole(g, (n, k), 82)
    down, up = _whole(g, (slots, rank, k), 82), _whole(g, (slots, n, rank), 82)
    live = torch.arange(rank, device=DEV) < torch.tensor(ranks, device=DEV)[:, None]
    down, up = down * live[:, :, None], up * live[:, None, :]
    order = torch.randperm(slots, generator=g, device=DEV)
    # the slots in an order of the seed's, with the ranks that belong to them
    down, up = down.index_select(0, order), up.index_select(0, order)
    host = order.tolist()
    place = [host.index(s) for s in range(slots)]
    scale = torch.randint(1024, 8192, (slots,), generator=g, device=DEV, dtype=torch.int32).to(torch.int16)
    per_row = [(-1 if a < 0 else place[a]) for a in _slots_of_requests(case) for _ in range(case["per"])][:rows]
    slot = torch.tensor(per_row, dtype=torch.int32, device=DEV)
    s = {"op": "project", "x": x, "slot": slot, "wide": case["wide"]}
    if own:
        llmx = _framework()
        stream = torch.cuda.current_stream().cuda_stream
        a = llmx.Adapters(k, n, w.data_ptr(), slots, rank, rows, stream=stream)
        scales = scale.tolist()
        for p in range(slots):
            r = ranks[host[p]]
            a.set(p, r, scales[p], down[p, :r].contiguous().data_ptr(), up[p, :, :r].contiguous().data_ptr(), stream=stream)
        torch.cuda.synchronize()  # the layouts are made: what they were made from may go
        s.update(llmx=llmx, plan=a, fmt=llmx.OUT_Q16_16 if case["wide"] else llmx.OUT_Q8_8,
                 out=torch.empty((rows, n), dtype=torch.int32 if case["wide"] else torch.int16, device=DEV))
    else:
        s.update(w=w, down=down, up=up, scale=scale)
    return s


def _logits(z):
    return (z * 65536).round_().clamp_(-(2.0**31) + 256, 2.0**31 - 256).to(torch.int32)


def _prepare_verify(case, g):
    b, k, v = case["requests"], case["drafts"], case["vocab"]
    counts = _counts(case)
    total = sum(counts)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    rows = total + b
    # peaked rows: a few likely tokens over a wide floor
    z = torch.randn((rows, v), generator=g, device=DEV) * 2.5
    likely = torch.randint(0, v, (rows, 12), generator=g, device=DEV)
    z.scatter_add_(1, likely, torch.rand((rows, 12), generator=g, device=DEV) * 14)
    owner = [q for q in range(b) for _ in range(counts[q])]
    target_row = torch.tensor([starts[q] + q + j for q in range(b) for j in range(counts[q])], dtype=torch.long, device=DEV)
    temperature = torch.rand((b,), generator=g, device=DEV) + 0.5
    temperature[1::7] = 0.0  # greedy requests among the others
    t_row = temperature[torch.tensor(owner, dtype=torch.long, device=DEV)].clamp_min(0.05) if total else None
    draft = None
    if total and case["model"]:
        dz = z[target_row] + torch.randn((total, v), generator=g, device=DEV) * 0.7
        tokens = torch.multinomial(torch.softmax(dz / t_row[:, None], 1), 1, generator=g)[:, 0]
        draft = _logits(dz)
        del dz
    elif total:
        tokens = torch.multinomial(torch.softmax(z[target_row], 1), 1, generator=g)[:, 0]
    else:
        tokens = torch.zeros((0,), dtype=torch.long, device=DEV)
    target = _logits(z)
    del z
    if case["ragged"]:  # tokens that a request's rules exclude
        target.masked_fill_(torch.rand((rows, v), generator=g, device=DEV) < 0.25, NONE)
    words = torch.randint(-(2**31), 2**31, (total + b,), generator=g, device=DEV).to(torch.int32)
    s = {"op": "verify", "target": target, "draft": draft, "tokens": tokens.to(torch.int32), "most": k,
         "offsets": torch.tensor(starts, dtype=torch.int32, device=DEV), "temperature": temperature,
         "accept": words[:total].contiguous(), "sample": words[total:].contiguous()}
    if own:
        llmx = _framework()
        size = llmx.verify_workspace_bytes(b, total, v)
        s.update(llmx=llmx, work=torch.empty((size,), dtype=torch.uint8, device=DEV),
                 out=torch.empty((b, k + 1), dtype=torch.int32, device=DEV),
                 accepted=torch.empty((b,), dtype=torch.int32, device=DEV),
                 probs=torch.empty((total, 2), dtype=torch.int64, device=DEV))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if s["op"] == "project":
        return _own_project(s) if own else _plain_project(s)
    return _own_verify(s) if own else _plain_verify(s)


def _own_project(s):
    x, out = s["x"], s["out"]
    s["plan"].project(x.data_ptr(), x.shape[0], s["slot"].data_ptr(), out.data_ptr(), s["fmt"],
                      stream=torch.cuda.current_stream().cuda_stream)
    return out


def _own_verify(s):
    target, draft, tokens = s["target"], s["draft"], s["tokens"]
    s["llmx"].verify_drafts(target.data_ptr(), draft.data_ptr() if draft is not None else None, target.shape[1],
                            tokens.data_ptr(), s["offsets"].data_ptr(), s["accepted"].shape[0], tokens.shape[0], s["most"],
                            s["temperature"].data_ptr(), s["accept"].data_ptr(), s["sample"].data_ptr(), s["out"].data_ptr(),
                            s["accepted"].data_ptr(), s["probs"].data_ptr(), s["work"].data_ptr(), s["work"].numel(),
                            stream=torch.cuda.current_stream().cuda_stream)
    return {"tokens": s["out"], "accepted": s["accepted"], "probs": s["probs"]}


def _rnd(v, k):
    return torch.floor(v / 2**k + 0.5)


def _plain_project(s):
    x, slot = s["x"].double(), s["slot"].long()
    y = x @ s["w"].double().T
    has = slot >= 0
    a = slot.clamp_min(0)
    t = torch.bmm(s["down"][a].double(), x.unsqueeze(2)).squeeze(2)
    t = _rnd(t * s["scale"][a].double().unsqueeze(1), 24).clamp_(-32768, 32767) * has.unsqueeze(1)
    # every slot's rows against its up matrix: t spread over the slots' columns
    slots, n, r = s["up"].shape
    wide = torch.zeros((x.shape[0], slots, r), dtype=torch.float64, device=x.device)
    wide[torch.arange(x.shape[0], device=x.device), a] = t
    y += wide.view(-1, slots * r) @ s["up"].permute(0, 2, 1).reshape(slots * r, n).double()
    q = _rnd(y, 4).clamp_(-(2.0**31), 2.0**31 - 1)
    return q.to(torch.int32) if s["wide"] else _rnd(q, 8).clamp_(-32768, 32767).to(torch.int16)


def weight(logits, temperature):
    """Whole-number softmax weights of rows of Q16.16 logits: 2^31 at the row's
    maximum, floor(2^31 2^-e) at e = (max - logit) log2(e) / T in 32-bit steps, 0
    where excluded; a temperature of at most 1e-6 leaves the first maximum alone."""
    z = logits.long()
    top = z.amax(1, keepdim=True)
    greedy = ~(temperature > 1e-6).unsqueeze(1)
    warm = torch.where(greedy, 1.0, temperature.unsqueeze(1))
    scale = torch.full_like(warm, LOG2E_16) / warm
    e = ((top - z).float() * scale).clamp_max_(100.0)
    i = torch.round(e)
    f = i - e
    p = f * COEF[4] + COEF[3]
    p = p * f + COEF[2]
    p = p * f + COEF[1]
    p = p * f + COEF[0]
    p = p * f + 1.0
    w = (p * 2.0**31).long() >> i.long().clamp_max(63)
    at = torch.arange(z.shape[1], device=z.device)
    first = torch.where(z == top, at, z.shape[1]).amin(1, keepdim=True)
    w = torch.where(greedy, (at == first).long() << 31, w)
    return w.masked_fill_(z == NONE, 0)


def _share(w):
    """Q0.40 probabilities of rows of weights."""
    total = w.sum(1, keepdim=True)
    # S >> h in [2^31, 2^32): the maximum's weight is 2^31, so h >= 0
    h = ((total >> torch.arange(32, 56, device=w.device)) > 0).sum(1, keepdim=True)
    inverse = (1 << 62) // (total >> h).clamp_min(1)
    return (w * inverse) >> (22 + h)


def _times(a, u):
    """floor(a u / 2^32) of whole numbers a < 2^45 and u < 2^32."""
    return (a * (u >> 16) + ((a * (u & 65535)) >> 16)) >> 16


def _plain_verify(s):
    offsets, tokens, most = s["offsets"].long(), s["tokens"].long(), s["most"]
    b, total, vocab = offsets.shape[0] - 1, tokens.shape[0], s["target"].shape[1]
    counts = offsets[1:] - offsets[:-1]
    dev = tokens.device
    requests = torch.arange(b, device=dev)
    owner = torch.repeat_interleave(requests, counts, output_size=total)
    row = torch.arange(total, device=dev) + owner  # each request has one target row more than drafts
    target_owner = torch.repeat_interleave(requests, counts + 1, output_size=total + b)
    p = _share(weight(s["target"], s["temperature"][target_owner]))
    q = _share(weight(s["draft"], s["temperature"][owner])) if s["draft"] is not None else None
    each = torch.arange(total, device=dev)
    p_token = p[row, tokens]
    q_token = q[each, tokens] if q is not None else torch.full_like(tokens, 1 << 40)
    passed = _times(q_token, s["accept"].long() & 0xFFFFFFFF) < p_token
    # the first rejection of each request
    j = each - offsets[owner]
    first = counts.clone().scatter_reduce_(0, owner, torch.where(passed, most + 1, j), "amin")
    at = offsets[:-1] + requests + first
    final = p[at]
    if total:
        drafted = (offsets[:-1] + first).clamp_max(total - 1)
        if q is not None:
            less = q[drafted]
        else:
            less = (torch.arange(vocab, device=dev) == tokens[drafted].unsqueeze(1)).long() << 40
        rest = (final - less).clamp_min_(0)
        use = ((first < counts) & (rest.sum(1) > 0)).unsqueeze(1)
        final = torch.where(use, rest, final)
    mass = final.cumsum(1)
    point = _times(mass[:, -1], s["sample"].long() & 0xFFFFFFFF)
    drawn = (mass <= point.unsqueeze(1)).sum(1)
    drawn = torch.where(mass[:, -1] > 0, drawn, -1)
    place = torch.arange(most + 1, device=dev)
    padded = torch.cat([tokens, tokens.new_full((1,), -1)])
    copied = padded[(offsets[:-1].unsqueeze(1) + place).clamp_max(total)]
    out = torch.where(place < first.unsqueeze(1), copied, -1)
    out = torch.where(place == first.unsqueeze(1), drawn.unsqueeze(1), out)
    return {"tokens": out.to(torch.int32), "accepted": first.to(torch.int32), "probs": torch.stack([p_token, q_token], 1)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "project":
        rows, k, n = case["rows"], case["k"], case["n"]
        ranks, reqs = _ranks(case), _slots_of_requests(case)
        used = sum(ranks[a] for a in set(reqs) if a >= 0)
        each = sum(ranks[a] for q, a in enumerate(reqs) if a >= 0 for _ in range(min(case["per"], rows - q * case["per"])))
        return {"bytes": 2 * n * k + 2 * rows * k + 4 * rows + 2 * used * (k + n) + rows * n * (4 if case["wide"] else 2),
                "flops": 2 * rows * n * k + 2 * each * (k + n)}
    counts = _counts(case)
    total, b, v = sum(counts), case["requests"], case["vocab"]
    rows = total + b + (total if case["model"] else 0)
    # a weight (17 operations) and a sum for each logit
    return {"bytes": 4 * rows * v + 24 * total + 16 * b + 4 * b * (case["drafts"] + 1), "flops": 18 * rows * v}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, on the host
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    h = {f: (v.cpu().numpy() if isinstance(v, torch.Tensor) else v) for f, v in s.items()}
    if case["op"] == "project":
        if case["rows"] * case["n"] * case["k"] > 2e9:
            return None
        return _exact_project(h)
    if (case["requests"] * (2 * case["drafts"] + 1)) * case["vocab"] > 6e6:
        return None
    return _exact_verify(h)


def _exact_project(h):
    x = h["x"].astype(np.float64)
    y = np.matmul(x, h["w"].astype(np.float64).T).astype(np.int64)  # below 2^53: exact
    for i, a in enumerate(h["slot"]):
        if a >= 0:
            t = np.matmul(h["down"][a].astype(np.float64), x[i]).astype(np.int64)
            t = np.clip((t * int(h["scale"][a]) + (1 << 23)) >> 24, -32768, 32767)
            y[i] += np.matmul(h["up"][a].astype(np.int64), t)
    q = np.clip((y + 8) >> 4, -(2**31), 2**31 - 1)
    return q.astype(np.int32) if h["wide"] else np.clip((q + 128) >> 8, -32768, 32767).astype(np.int16)


def _exact_row(z, temperature):
    """Q0.40 probabilities of one row, as Python's whole numbers."""
    z = z.astype(np.int64)
    top = int(z.max())
    if top == NONE:
        return np.zeros(len(z), np.int64)
    if not temperature > 1e-6:
        w = np.zeros(len(z), np.int64)
        w[int(np.argmax(z))] = 1 << 31
    else:
        f32 = np.float32
        scale = f32(LOG2E_16) / f32(temperature)
        e = np.minimum((top - z).astype(f32) * scale, f32(100))
        i = np.rint(e)
        f = i - e
        g = f * f32(COEF[4]) + f32(COEF[3])
        for c in (COEF[2], COEF[1], COEF[0], 1.0):
            g = g * f + f32(c)
        w = np.floor(np.ldexp(g.astype(np.float64), 31 - i.astype(np.int64))).astype(np.int64)
        w[z == NONE] = 0
    total = int(w.sum())
    h = total.bit_length() - 32
    inverse = (1 << 62) // (total >> h)
    return (w * inverse) >> (22 + h)


def _exact_verify(h):
    b, most = len(h["offsets"]) - 1, h["most"]
    out = np.full((b, most + 1), -1, np.int32)
    accepted, probs = np.zeros(b, np.int32), np.zeros((len(h["tokens"]), 2), np.int64)
    for r in range(b):
        at, count = int(h["offsets"][r]), int(h["offsets"][r + 1] - h["offsets"][r])
        n, stopped, less = 0, False, None
        for j in range(count):
            x = int(h["tokens"][at + j])
            p = _exact_row(h["target"][at + r + j], h["temperature"][r])
            if h["draft"] is not None:
                q = _exact_row(h["draft"][at + j], h["temperature"][r])
            else:
                q = np.zeros(len(p), np.int64)
                q[x] = 1 << 40
            probs[at + j] = p[x], q[x]
            if not stopped and int(h["accept"][at + j]) % 2**32 * int(q[x]) < int(p[x]) << 32:
                out[r, j] = x
                n += 1
            elif not stopped:
                stopped, less = True, np.maximum(p - q, 0)
        p = _exact_row(h["target"][at + r + n], h["temperature"][r])
        if stopped and less.sum() > 0:
            p = less
        mass = np.cumsum(p)
        point = int(h["sample"][r]) % 2**32 * int(mass[-1]) >> 32
        out[r, n] = int(np.searchsorted(mass, point, side="right")) if mass[-1] else -1
        accepted[r] = n
    return {"tokens": out, "accepted": accepted, "probs": probs}
