"""A batch of sessions behind one system prompt, decoded speculatively from an 8-bit paged cache.

One step, as a server runs it: every session drafts tokens by looking up what followed its last token
before; the drafted rows' K and V are quantised into the sessions' pages (kvq_write); all rows attend the
shared prompt, held once for all, and their own pages (kvq_attention); the target's probabilities accept
or refuse the drafts and give the next token (verify_draft); refused positions are dropped by the length
alone.  The model is one random attention layer, so that the example needs no checkpoint.

    python examples/speculative_serving.py --batch 8 --drafts 4 --steps 32
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from dotllm_b200 import serving  # noqa: E402


class OneLayer:
    """Random embedding, positions, one attention layer and a head; fp32 activations."""

    def __init__(self, vocab=512, hidden=256, heads=8, heads_kv=2, head_dim=64, positions=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def rand(*shape, scale=1.0):
            return torch.randn(*shape, device="cuda", generator=g) * scale

        self.vocab, self.heads, self.heads_kv, self.head_dim = vocab, heads, heads_kv, head_dim
        self.embed, self.position = rand(vocab, hidden), rand(positions, hidden, scale=0.1)
        self.head = rand(hidden, vocab, scale=4.0 * hidden ** -0.5)
        self.qkv = rand(hidden, (heads + 2 * heads_kv) * head_dim, scale=hidden ** -0.5)
        self.out = rand(heads * head_dim, hidden, scale=(heads * head_dim) ** -0.5)

    def project(self, tokens, positions):
        """q [rows, heads, dim], k and v [rows, heads_kv, dim]: slices of one product."""
        x = self.embed[tokens] + self.position[positions]
        y = (x @ self.qkv).view(len(tokens), -1, self.head_dim)
        return x, y[:, :self.heads], y[:, self.heads:self.heads + self.heads_kv], y[:, self.heads + self.heads_kv:]

    def logits(self, x, attended):
        return (x + attended.flatten(1) @ self.out) @ self.head


def lookup_draft(history, count):
    """The tokens that followed the latest earlier occurrence of the last one (or the last one again)."""
    last = history[-1]
    for i in range(len(history) - 2, -1, -1):
        if history[i] == last:
            found = history[i + 1:i + 1 + count]
            return found + [last] * (count - len(found))
    return [last] * count


def serve(model, prompt, first, steps, drafts, cache=torch.int8, greedy=False, seed=1):
    """`steps` steps for len(first) sessions that continue `prompt` with one own token each.  Returns the sessions'
    tokens and the number of drafts accepted."""
    B, k, P = len(first), drafts, len(prompt)
    own_pages = -(-(1 + steps * (k + 1) + k) // serving.PAGE)
    prefix_pages = -(-P // serving.PAGE)
    pool = serving.KvqPool.empty(prefix_pages + B * own_pages, model.heads_kv, model.head_dim, cache)
    ids = torch.randperm(prefix_pages + B * own_pages, device="cuda", dtype=torch.int32)
    prefix, pages = ids[:prefix_pages], ids[prefix_pages:].view(B, own_pages)
    i32 = dict(dtype=torch.int32, device="cuda")
    # the prompt's K and V, once for all sessions
    at = torch.arange(P, device="cuda")
    _, _, pk, pv = model.project(torch.tensor(prompt, device="cuda"), at)
    serving.kvq_write(pool, serving.KvqBatch(torch.tensor([0, P], **i32), torch.tensor([P], **i32), prefix.view(1, -1), P), pk, pv)

    rows = k + 1
    row_start = torch.arange(B + 1, **i32) * rows
    seq_len = torch.zeros(B, **i32)  # positions whose K and V are settled
    batch = serving.KvqBatch(row_start, seq_len, pages, rows)
    g = torch.Generator(device="cuda").manual_seed(seed)
    texts, accepted_all = [[t] for t in first], 0
    for _ in range(steps):
        draft = torch.tensor([lookup_draft(prompt + t, k) for t in texts], **i32).view(B, k)
        last = torch.tensor([[t[-1]] for t in texts], **i32)
        tokens = torch.cat([last, draft], 1).flatten()
        seq_len += rows  # the rows are the sequences' last positions
        place = (P + seq_len.long()[:, None] - rows + torch.arange(rows, device="cuda")).flatten()
        x, q, key, value = model.project(tokens, place)
        serving.kvq_write(pool, batch, key, value)
        y = serving.kvq_attention(pool, batch, q, prefix_pages=prefix, prefix_len=P)
        logits = model.logits(x, y).view(B, rows, model.vocab)
        if greedy:  # the target's distribution is its argmax
            p = torch.zeros_like(logits).scatter_(2, logits.argmax(-1, keepdim=True), 1.0)
        else:
            p = torch.softmax(logits, -1)
        uniform = torch.rand(B, rows, device="cuda", generator=g)
        out, accepted = serving.verify_draft(p, None, draft, uniform)  # looked-up drafts have no probabilities
        seq_len -= k - accepted  # refused positions are written over by the next step
        for t, new in zip(texts, out.tolist()):
            t += [n for n in new if n >= 0]
        accepted_all += int(accepted.sum())
    return texts, accepted_all


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--cache", choices=["int8", "e4m3"], default="int8")
    ap.add_argument("--greedy", action="store_true")
    a = ap.parse_args()
    model = OneLayer()
    g = torch.Generator().manual_seed(7)
    prompt = torch.randint(0, model.vocab, (a.prompt,), generator=g).tolist()
    first = torch.randint(0, model.vocab, (a.batch,), generator=g).tolist()
    texts, accepted = serve(model, prompt, first, a.steps, a.drafts, torch.int8 if a.cache == "int8" else torch.float8_e4m3fn, a.greedy)
    made = sum(len(t) - 1 for t in texts)
    print(f"{a.batch} sessions, {a.steps} steps: {made} tokens, {accepted} of {a.batch * a.steps * a.drafts} drafts accepted")
    print("session 0:", texts[0][:24])


if __name__ == "__main__":
    main()
