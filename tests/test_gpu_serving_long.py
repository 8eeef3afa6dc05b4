"""Shared-prefix attention over many pages and many rows, against a dense 64-bit form on the device: what the
small cases of test_gpu_serving.py do not reach -- pipelines that wrap round their stages many times,
references that have to rise in the middle, value scales that grow, prompt chunks of hundreds of rows.

Bars as in test_gpu_serving.py: with X the largest sum |q_i k_i| scale of a row, e = 2^-21 X is what a score
may be off by, hence the output by 2 e V (V the largest |v|), plus 2^-18 V for the sums over the positions,
2^-11 V for weights rounded to 11 bits and the output's own rounding (2^-11 V fp16, 2^-8 V bf16).
"""
import pytest

pytestmark = pytest.mark.gpu
PAGE = 64
ROUND = {"f32": 0.0, "f16": 2.0 ** -11 + 2.0 ** -11, "bf16": 2.0 ** -11 + 2.0 ** -8}


def quantise(x, fmt):
    import torch
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "i8":
        return torch.round(x * (127.0 / top)).clamp(-127, 127).to(torch.int8), (top / 127.0).squeeze(-1)
    return (x * (448.0 / top)).clamp(-448, 448).to(torch.float8_e4m3fn), (top / 448.0).squeeze(-1)


def run(fmt, typ, hk, group, dim, prefix, lens, rows, window=0, softcap=0.0, k_ramp=0.0, v_ramp=0.0, scale=None, q_scale=1.0, seed=0):
    """k_ramp, v_ramp: K and V grow by that many powers of two from the first position to the last."""
    import torch
    from dotllm_b200 import serving
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    g = torch.Generator("cuda").manual_seed(seed)
    B, R = len(lens), sum(rows)
    need = [-(-n // PAGE) for n in lens]
    npre, most = -(-prefix // PAGE), max(need + [1])
    total = npre + sum(need) + 1
    ids = torch.randperm(total, device="cuda", generator=g).int()
    table = torch.full((B, most), -1, dtype=torch.int32, device="cuda")
    at = npre
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    parts, values = [], []
    for ramp in (k_ramp, v_ramp):
        codes = torch.full((total, hk, PAGE, dim), -1, dtype=torch.int8, device="cuda")
        scales = torch.full((total, hk, PAGE), float("nan"), device="cuda")
        held = []
        for n, pages, first in [(prefix, ids[:npre], 0)] + [(lens[b], table[b], prefix) for b in range(B)]:
            j = torch.arange(n, device="cuda")
            x = torch.randn(n, hk, dim, device="cuda", generator=g) * torch.exp2(ramp * (first + j) / max(1, prefix + max(lens + [1])))[:, None, None]
            c, s = quantise(x, fmt)
            codes[pages[j // PAGE].long(), :, j % PAGE] = c.view(torch.int8)
            scales[pages[j // PAGE].long(), :, j % PAGE] = s
            held.append(c.double() * s.double()[..., None])
        parts += [codes.view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn), scales]
        values.append(held)
    pool = serving.KvqPool(parts[0], parts[2], parts[1], parts[3])
    row_start = torch.tensor([0] + rows, device="cuda").cumsum(0).int()
    batch = serving.KvqBatch(row_start, torch.tensor(lens, dtype=torch.int32, device="cuda"), table, max(rows))
    q = (torch.randn(R, hk * group, dim, device="cuda", generator=g) * q_scale).to(types[typ])
    out, lse = serving.kvq_attention(pool, batch, q, prefix_pages=ids[:npre].contiguous(), prefix_len=prefix, window=window,
                                     softcap=softcap, scale=scale, return_lse=True)
    sc = dim ** -0.5 if scale is None else scale
    r = 0
    for b in range(B):
        n, T = rows[b], prefix + lens[b]
        k = torch.cat([values[0][0], values[0][1 + b]]).transpose(0, 1)  # [hk, T, dim]
        v = torch.cat([values[1][0], values[1][1 + b]]).transpose(0, 1)
        x = q[r:r + n].double().view(n, hk, group, dim).permute(1, 0, 2, 3).reshape(hk, n * group, dim)
        s = x @ k.transpose(1, 2) * sc
        big = float((x.abs() @ k.abs().transpose(1, 2)).max()) * abs(sc)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p = T - n + torch.arange(n, device="cuda").repeat_interleave(group)[:, None]
        j = torch.arange(T, device="cuda")[None]
        s = s.masked_fill((j > p) | (j <= p - (window or T + n)), float("-inf"))
        want_lse = torch.logsumexp(s, -1)
        want = torch.exp(s - want_lse[..., None]) @ v
        got = out[r:r + n].double().view(n, hk, group, dim).permute(1, 0, 2, 3).reshape(hk, n * group, dim)
        got_lse = lse[r:r + n].double().view(n, hk, group).permute(1, 0, 2).reshape(hk, n * group)
        V = float(v.abs().max())
        e = 2.0 ** -21 * big
        assert torch.isfinite(got).all()
        err = float((got - want).abs().max())
        assert err <= (2 * e + 2.0 ** -18 + ROUND[typ]) * V, (b, err, V)
        assert ((got_lse - want_lse).abs() <= e + 2.0 ** -20 * (1 + want_lse.abs())).all()
        r += n
    return out


@pytest.mark.parametrize("typ", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (96, "e4m3"), (128, "i8"), (256, "e4m3")])
@pytest.mark.parametrize("k_ramp,v_ramp", [(0.0, 0.0), (5.0, 8.0)])
def test_long_prefix_many_rows(gpu, typ, dim, fmt, k_ramp, v_ramp):
    """Sixteen pages and more per CTA; with the ramps the scores' maximum and the values' scale rise all along."""
    rows = [1 + i % 4 for i in range(52)]
    run(fmt, typ, 32, 2, dim, 2010, [r + 5 * i for i, r in enumerate(rows)], rows, k_ramp=k_ramp, v_ramp=v_ramp, q_scale=0.5)


@pytest.mark.parametrize("typ", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("window", [0, 100])
def test_prompt_chunks(gpu, typ, dim, window):
    """Chunks of hundreds of rows of one sequence (masks in every tile), with and without earlier positions."""
    run("i8", typ, 2, 3, dim, 70, [300, 129, 64], [300, 100, 1], window=window)
    run("e4m3", typ, 1, 4, dim, 0, [257], [257], window=window, softcap=8.0, q_scale=3.0)


@pytest.mark.parametrize("typ", ["f16", "bf16", "f32"])
def test_long_sequences_few_rows(gpu, typ):
    """Long own caches, chunks of many pages, references that rise; a negative scale."""
    run("i8", typ, 2, 4, 128, 0, [20000, 3, 7777], [1, 2, 5], k_ramp=4.0, v_ramp=6.0)
    run("e4m3", typ, 8, 1, 64, 5000, [6000] * 3, [1, 1, 1], k_ramp=4.0, scale=-0.2)
    run("i8", typ, 2, 2, 128, 300, [200] * 40, [1] * 40, scale=-0.1, window=333)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_many_rows_from_unaligned_queries(gpu, typ):
    """Queries that start off every 16-byte boundary, and rows strided as slices of a wider product, give the bits
    that dense ones give."""
    import torch
    from dotllm_b200 import serving
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[typ]
    g = torch.Generator("cuda").manual_seed(3)
    R, hk, heads, dim, P = 90, 2, 4, 128, 500
    pool = serving.KvqPool.empty(8, hk, dim)
    rows = torch.tensor([0, P], dtype=torch.int32, device="cuda")
    pages = torch.arange(8, dtype=torch.int32, device="cuda")
    serving.kvq_write(pool, serving.KvqBatch(rows, rows[1:].contiguous(), pages.view(1, -1), P),
                      torch.randn(P, hk, dim, device="cuda", generator=g), torch.randn(P, hk, dim, device="cuda", generator=g))
    batch = serving.KvqBatch(torch.arange(R + 1, dtype=torch.int32, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda"),
                             torch.full((R, 1), -1, dtype=torch.int32, device="cuda"), 1)
    flat = torch.randn(R * 6 * dim + 1, device="cuda", generator=g).to(t)
    for wide in (flat[1:].view(R, 6, dim), flat[:-1].view(R, 6, dim)):
        q = wide[:, 1:5]
        a = serving.kvq_attention(pool, batch, q, prefix_pages=pages, prefix_len=P)
        b = serving.kvq_attention(pool, batch, q.contiguous(), prefix_pages=pages, prefix_len=P)
        # a sequence of length 0 puts its row just before its own first position: it sees the whole prefix
        assert torch.equal(a, b) and bool((a != 0).any())


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (96, "e4m3"), (128, "i8"), (256, "e4m3")])
@pytest.mark.parametrize("hk,prefix,lens,rows", [
    (2, 1000, [333], [9]),               # 18 rows: prefix and own pages may go to different kernels
    (2, 130, [700, 20], [12, 1]),        # 24 own rows, 26 on the prefix
    (1, 0, [2900, 64, 65], [8, 9, 17]),  # 34 own rows at most, no prefix
    (2, 6400, [8], [8]),                 # 16 rows
    (32, 4500, [400, 1, 90], [10, 1, 3]),  # many heads: 28 rows on more pages
])
def test_middling_rows(gpu, typ, dim, fmt, hk, prefix, lens, rows):
    """8 to 34 rows of a kv head (two query heads each), on either side of where the kernels change."""
    run(fmt, typ, hk, 2, dim, prefix, lens, rows, window=0, q_scale=0.7)
    run(fmt, typ, hk, 2, dim, prefix, lens, rows, window=150, softcap=20.0, k_ramp=3.0, v_ramp=3.0)
