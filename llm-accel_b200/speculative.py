"""Several requests at once, each with its own low-rank adapter, decoded with
drafts that one call verifies for all of them.

The step of a serving loop: every request runs its last token and its drafts as
one block through its decoder stack (llmx_stack_async, up to 8 rows), the
final-normed rows of all requests go through the LM head together, each with
its request's adapter (llmx_adapters_project, Q16.16 logits), and the drafts are
verified and a next token drawn for all of them (llmx_verify_drafts).  Drafts are
copied from the request's own text: what followed the last two tokens
when they last occurred.  Rows of rejected drafts leave nothing behind: the next block
starts at the first position that was not accepted and overwrites their K/V.

Every request has a context, so a K/V cache, of its own; the contexts hold
the same weights.  Needs torch for the device arrays.
"""
from __future__ import annotations

import numpy as np

import llmx

NO_TOKEN = 0xFFFFFFFF


def copied_drafts(tokens, most):
    """What followed the last earlier occurrence of the last two tokens, at most `most` tokens."""
    for at in range(len(tokens) - 3, -1, -1):
        if tokens[at:at + 2] == tokens[-2:]:
            return tokens[at + 2:at + 2 + most]
    return []


def append_tokens(texts, goal, tokens, accepted):
    """Appends a step's tokens [requests][most + 1] to the texts that are short of their goal, and says
    how many drafts were accepted for them; raises, with the texts as they were, where the verification
    has no tokens for a request (accepted = 0xffffffff) or no token could be drawn."""
    words = lambda a: np.ascontiguousarray(a).view(np.uint32)  # noqa: E731
    tokens, accepted = words(tokens), words(accepted)
    new = {}
    for r, text in enumerate(texts):
        if len(text) >= goal[r]:
            continue
        if accepted[r] >= tokens.shape[1]:
            raise llmx.LlmxError(llmx.ERR_TIMEOUT, f"request {r}: the verification gave up")
        new[r] = tokens[r, :accepted[r] + 1].tolist()
        if NO_TOKEN in new[r]:
            raise llmx.LlmxError(llmx.ERR_RANGE, f"request {r}: its row excludes every token")
    for r, more in new.items():
        texts[r] += more
    return sum(len(more) - 1 for more in new.values())


class Server:
    def __init__(self, model: llmx.Model, requests, slots, max_rank, drafts=4, device=0):
        import torch

        if not 0 <= drafts < llmx.MAX_ROWS:
            raise ValueError("drafts must be 0..7: a block has the last token and the drafts")
        self.torch, self.model, self.s = torch, model, model.shape
        self.dev, self.drafts = torch.device("cuda", device), drafts
        self.contexts = [llmx.Accelerator(self.s, device) for _ in range(requests)]
        for c in self.contexts:
            c.upload_model(model)
        # the handle keeps its own layout of the LM head.  An LM head is Q4.12; an embedding that
        # stands in for it is Q8.8, so that what the handle writes as Q16.16 is 1/16 of the logits
        table = torch.from_numpy(model.lm_head()).to(self.dev)
        self.logit_step = 16.0 if model.tied else 1.0
        self.rows = requests * (drafts + 1)
        self.head = llmx.Adapters(self.s.hidden, self.s.vocab, table.data_ptr(), slots, max_rank, self.rows, device,
                                  stream=self.stream())
        new = lambda shape, kind: torch.zeros(shape, dtype=kind, device=self.dev)  # noqa: E731
        self.x = new((self.rows, self.s.hidden), torch.int16)
        self.logits = new((self.rows, self.s.vocab), torch.int32)
        self.tokens, self.accepted = new((requests, drafts + 1), torch.int32), new((requests,), torch.int32)
        size = llmx.verify_workspace_bytes(requests, requests * drafts, self.s.vocab)
        self.work = new((size,), torch.uint8)
        torch.cuda.synchronize(self.dev)

    def close(self):
        self.head.close()
        for c in self.contexts:
            c.close()

    def stream(self):
        return self.torch.cuda.current_stream(self.dev).cuda_stream

    def set_adapter(self, slot, scale, down, up):
        """down [rank][hidden] and scale: Q4.12; up [vocab][rank]: in the LM head's format
        (Q4.12, or Q8.8 where the embedding stands in for it)."""
        down, up = np.asarray(down), np.asarray(up)
        if down.ndim != 2 or up.shape != (self.s.vocab, len(down)) or down.shape[1] != self.s.hidden:
            raise ValueError(f"down {down.shape} and up {up.shape} are not [rank][{self.s.hidden}] and [{self.s.vocab}][rank]")
        for what, a in (("down", down), ("up", up), ("scale", np.asarray(scale))):
            if a.dtype.kind not in "iu" or (a.size and (a.min() < -32768 or a.max() > 32767)):
                raise ValueError(f"{what} is not whole numbers of 16 bits")
        d, u = (self.torch.from_numpy(np.ascontiguousarray(a, np.int16)).to(self.dev) for a in (down, up))
        self.head.set(slot, d.shape[0], scale, d.data_ptr(), u.data_ptr(), stream=self.stream())
        self.torch.cuda.current_stream(self.dev).synchronize()

    def _block(self, request, tokens, position, row):
        """Runs a block of one request; its final-normed rows go to x[row:]."""
        c, n = self.contexts[request], len(tokens)
        c.write_hidden(1, self.model.embed(tokens))
        c.stack_async(n, 0, self.s.layers, position)
        here = self.torch.cuda.current_stream(self.dev)
        here.wait_stream(self.torch.cuda.ExternalStream(c.stream, device=self.dev))
        self.x[row:row + n].view(-1).copy_(_view(self.torch, c.hidden_ptr(0), n * self.s.hidden, self.dev))

    def generate(self, prompts, slots, max_new, temperature=0.0, seed=0):
        """New tokens of every request, and (drafted, accepted) over all of them."""
        t, count = self.torch, len(prompts)
        if count != len(self.contexts):
            raise ValueError(f"{count} prompts for {len(self.contexts)} requests")
        if len(slots) != count:
            raise ValueError(f"{len(slots)} slots for {count} requests")
        if any(len(p) == 0 for p in prompts):
            raise ValueError("a prompt has at least one token")
        rng = np.random.default_rng(seed)
        texts = [list(map(int, p)) for p in prompts]
        for r, text in enumerate(texts):  # all but the last prompt token
            for at in range(0, len(text) - 1, llmx.MAX_ROWS):
                block = text[at:min(at + llmx.MAX_ROWS, len(text) - 1)]
                self.contexts[r].stack(self.model.embed(block), position=at, include_final_norm=False, materialize=False)
        goal = [len(p) + max_new for p in prompts]
        dev = lambda a: t.from_numpy(np.ascontiguousarray(a).view(np.int32)).to(self.dev)  # noqa: E731
        temperatures = t.full((count,), float(temperature) / self.logit_step, device=self.dev)
        drafted = taken = 0
        while any(len(x) < g for x, g in zip(texts, goal)):
            guesses, offsets, row, owners = [], [0], 0, []
            for r, text in enumerate(texts):
                room = min(self.drafts, goal[r] - len(text) - 1)  # a request that is done runs along undrafted
                guess = copied_drafts(text, room) if room > 0 else []
                self._block(r, [text[-1]] + guess, len(text) - 1, row)
                row += 1 + len(guess)
                owners += [slots[r]] * (1 + len(guess))
                guesses += guess
                offsets.append(len(guesses))
            words = rng.integers(0, 2**32, len(guesses) + count, dtype=np.uint64).astype(np.uint32)
            d_owner, d_guess, d_offsets = dev(np.array(owners, np.int32)), dev(np.array(guesses, np.uint32)), dev(np.array(offsets, np.uint32))
            d_accept, d_sample = dev(words[:len(guesses)]), dev(words[len(guesses):])
            p = lambda a: a.data_ptr() if a.numel() else None  # noqa: E731
            self.head.project(self.x.data_ptr(), row, p(d_owner), self.logits.data_ptr(), llmx.OUT_Q16_16, stream=self.stream())
            llmx.verify_drafts(self.logits.data_ptr(), None, self.s.vocab, p(d_guess), p(d_offsets), count, len(guesses), self.drafts,
                               p(temperatures), p(d_accept), p(d_sample), p(self.tokens), p(self.accepted), None, p(self.work),
                               self.work.numel(), stream=self.stream())
            # nothing is made of rows or logits that a kernel gave up
            self.head.error(self.stream())
            for c in self.contexts:
                c.synchronize()
            drafted += sum(offsets[r + 1] - offsets[r] for r, text in enumerate(texts) if len(text) < goal[r])
            taken += append_tokens(texts, goal, self.tokens.cpu().numpy(), self.accepted.cpu().numpy())
        return [text[len(q):] for text, q in zip(texts, prompts)], (drafted, taken)


def _view(torch, pointer, count, device):
    """`count` int16 of a context's memory as a tensor, without a copy."""
    class Memory:
        __cuda_array_interface__ = {"shape": (count,), "typestr": "<i2", "data": (pointer, False), "version": 2}

    return torch.as_tensor(Memory(), device=device)


def main():
    """Three requests of the "small" profile, two with adapters: the tokens with and
    without drafts, which are the same ones (greedy)."""
    s = llmx.shape("small")
    model = llmx.Model(s).init_reference_random(7)
    rng = np.random.default_rng(1)
    prompts, slots = [[3, 9, 4, 3, 9], [5, 5, 5, 5], [1, 2, 3, 1, 2, 3, 1]], [0, -1, 1]
    for drafts in (0, 4):
        server = Server(model, 3, 2, 8, drafts)
        noise = np.random.default_rng(2)
        for slot, rank in ((0, 8), (1, 3)):
            server.set_adapter(slot, 4096, noise.integers(-400, 400, (rank, s.hidden)), noise.integers(-400, 400, (s.vocab, rank)))
        out, (drafted, taken) = server.generate(prompts, slots, 12, seed=int(rng.integers(1 << 30)))
        print(f"{drafts} drafts: {out}; {taken} of {drafted} drafts accepted")
        server.close()


if __name__ == "__main__":
    main()
