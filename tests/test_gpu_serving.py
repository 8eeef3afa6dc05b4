"""Serving operators on the device against plain 64-bit implementations: the 8-bit paged KV pool, the
shared-prefix attention over it, and the verification of drafted tokens.

Bars.  Codes, scales, values read back, tokens and counts: exact.  Attention: with e = 2^-21 X, X the
largest sum |q_i k_i| scale of a row (fp32 products summed in any order over at most 256 terms, the
exponential's error included), a score is off by at most e, hence the softmax weights by at most a
factor 1 + 2 e and the output by 2 e V, V the largest |v|; fp32 sums over the positions add 2^-18 V.
16-bit activations add the rounding of the weights to 11 bits, 2^-11 V, and of the output, half a unit
in the last place of V.  lse: e + 2^-20 (1 + |lse|).
"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PAGE = 64
TOP = {"i8": 127.0, "e4m3": 448.0}


def _torch():
    import torch
    return torch


def _types():
    t = _torch()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}


def _code_type(fmt):
    t = _torch()
    return t.int8 if fmt == "i8" else t.float8_e4m3fn


def quantise(x, fmt):
    """The definition, one IEEE fp32 operation at a time (CPU)."""
    t = _torch()
    x = x.float().cpu().numpy()
    a = np.abs(x).max(-1, keepdims=True)
    fine = np.isfinite(x).all(-1, keepdims=True)
    some = fine & (a >= np.float32(1e-30))
    M = np.float32(TOP[fmt])
    with np.errstate(all="ignore"):
        y = np.where(some, x * (M * (np.float32(1) / a)), np.float32(0)).astype(np.float32)
        scale = np.where(some, a / M, np.where(fine, np.float32(0), np.float32("nan"))).astype(np.float32)[..., 0]
    y = t.from_numpy(np.clip(y, -M, M))
    return (t.round(y).to(t.int8) if fmt == "i8" else y.to(t.float8_e4m3fn)), t.from_numpy(scale)


class Case:
    """A pool whose unused slots hold garbage, sequences on shuffled pages, and one call's rows."""

    def __init__(self, fmt, hk, dim, lens, rows, prefix=0, seed=0, spare=2, extra_pages=1, v_spread=0.0, base_page=0, n_pages=None):
        t = _torch()
        rng = np.random.default_rng(seed)
        need = [-(-n // PAGE) for n in lens]
        npre = -(-prefix // PAGE)
        used = sum(need) + npre
        n_pages = n_pages or used + spare
        ids = base_page + rng.permutation(n_pages - base_page)[:used]
        self.fmt, self.hk, self.dim, self.lens, self.rows, self.prefix = fmt, hk, dim, lens, rows, prefix
        most = max(need + [0]) + extra_pages
        table = np.full((len(lens), most), -1, np.int32)  # unused entries are no page
        at = npre
        self.prefix_ids = ids[:npre].astype(np.int32)
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            at += n
        self.table = table
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        shape = (n_pages, hk, PAGE, dim)
        self.kv = []  # values of K and V by (list, position): the prefix is list -1
        dev = []
        for which in range(2):
            codes = t.full(shape, -1, dtype=t.int8, device="cuda")  # 0xFF: -1, or a NaN as e4m3
            scales = t.full(shape[:3], float("nan"), device="cuda")
            vals = {}
            for b, (n, pages) in [(-1, (prefix, self.prefix_ids))] + [(b, (lens[b], table[b])) for b in range(len(lens))]:
                x = rng.standard_normal((n, hk, dim)).astype(np.float32)
                if which == 1 and v_spread:
                    x *= np.exp2(rng.uniform(-v_spread, 0, (n, hk, 1))).astype(np.float32)
                c, s = quantise(t.from_numpy(x), fmt)
                vals[b] = (c.float().numpy().astype(np.float64) * s.numpy().astype(np.float64)[..., None])
                if n:
                    j = np.arange(n)
                    p = t.from_numpy(pages[j // PAGE].astype(np.int64)).cuda()
                    o = t.from_numpy(j % PAGE).cuda()
                    codes[p, :, o] = c.view(t.int8).cuda()
                    scales[p, :, o] = s.cuda()
            self.kv.append(vals)
            dev += [codes.view(_code_type(fmt)), scales]
        from dotllm_b200 import serving
        self.pool = serving.KvqPool(dev[0], dev[2], dev[1], dev[3])
        self.batch = serving.KvqBatch(t.from_numpy(self.row_start).cuda(), t.tensor(lens, dtype=t.int32).cuda(),
                                      t.from_numpy(table).cuda(), max(list(rows) + [0]))
        self.prefix_pages = t.from_numpy(self.prefix_ids).cuda()

    def attend(self, q, **kw):
        from dotllm_b200 import serving
        return serving.kvq_attention(self.pool, self.batch, q, prefix_pages=self.prefix_pages, prefix_len=self.prefix,
                                     return_lse=True, **kw)

    def reference(self, q, window=0, softcap=0.0, hidden=()):
        """(out, lse, largest sum |q k| scale, largest |v|) in 64 bits; hidden: (sequence, position) never seen."""
        q = q.double().cpu().numpy()
        R, H, D = q.shape
        G = H // self.hk
        out, lse, X, Vm = np.zeros((R, H, D)), np.full((R, H), -np.inf), 0.0, 0.0
        r = 0
        for b, n in enumerate(self.rows):
            k = np.concatenate([self.kv[0][-1], self.kv[0][b]])
            v = np.concatenate([self.kv[1][-1], self.kv[1][b]])
            total = self.prefix + self.lens[b]
            gone = [self.prefix + j for (bb, j) in hidden if bb == b]
            for i in range(n):
                p = total - n + i
                js = np.arange(max(0, p - window + 1) if window else 0, max(p + 1, 0))
                js = np.setdiff1d(js, gone)
                if js.size:
                    for h in range(H):
                        kk, vv = k[js, h // G], v[js, h // G]
                        s = kk @ q[r, h] * D ** -0.5
                        X = max(X, (np.abs(kk) @ np.abs(q[r, h])).max() * D ** -0.5)
                        Vm = max(Vm, np.abs(vv).max())
                        if softcap:
                            s = softcap * np.tanh(s / softcap)
                        m = s.max()
                        e = np.exp(s - m)
                        lse[r, h] = m + np.log(e.sum())
                        out[r, h] = e @ vv / e.sum()
                r += 1
        return out, lse, X, Vm


def check_attention(c, q, typ, **kw):
    hidden = kw.pop("hidden", ())
    out, lse = c.attend(q, **kw)
    ref, rlse, X, V = c.reference(q, hidden=hidden, **kw)
    e = 2.0 ** -21 * X
    tol = 2 * e * V + 2.0 ** -18 * V
    if typ == "f16":
        tol += 2.0 ** -11 * V + 2.0 ** -11 * V
    if typ == "bf16":
        tol += 2.0 ** -11 * V + 2.0 ** -8 * V
    got, glse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert out.dtype == q.dtype and np.isfinite(got).all()
    assert np.array_equal(np.isinf(glse), np.isinf(rlse))
    err = np.abs(got - ref).max() if got.size else 0.0
    assert err <= tol, f"output off by {err}, {tol} allowed"
    seen = ~np.isinf(rlse)
    assert (np.abs(glse[seen] - rlse[seen]) <= e + 2.0 ** -20 * (1 + np.abs(rlse[seen]))).all()
    assert (got[~seen] == 0).all()
    return out, lse


def rand_q(R, H, D, typ, seed=0, scale=1.0):
    t = _torch()
    g = t.Generator().manual_seed(seed)
    return (t.randn(R, H, D, generator=g) * scale).to(_types()[typ]).cuda()


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("hk,dim,lens,rows", [
    (8, 64, [1], [1]), (2, 96, [64, 65, 1, 130], [1, 1, 1, 1]), (3, 128, [70, 200], [70, 131]),
    (1, 256, [63, 0, 5], [2, 0, 5]), (32, 96, [129] * 5, [3, 1, 0, 7, 129]), (5, 64, [3, 100], [5, 100])])
def test_write_and_read_back(gpu, typ, fmt, hk, dim, lens, rows):
    """Codes and scales equal the definition's, other slots stay, and reading returns code * scale rounded once.
    The last case has more rows than positions: those rows are written nowhere and read as zeros."""
    t = _torch()
    from dotllm_b200 import serving
    c = Case(fmt, hk, dim, lens, rows, seed=3)
    R = sum(rows)
    g = t.Generator().manual_seed(5)
    x = [(t.randn(R, hk, dim, generator=g) * t.exp(2 * t.randn(R, hk, 1, generator=g))).to(_types()[typ]) for _ in range(2)]
    x[0][0, 0] = 0
    x[1][0, 0, 0] = 1e-33 if typ == "f32" else 0
    if R > 2:
        x[0][1, 0, 7] = float("nan")
        x[1][2, hk - 1, dim - 1] = float("-inf")
    want = []
    for which, (codes, scales) in enumerate([(c.pool.k, c.pool.k_scale), (c.pool.v, c.pool.v_scale)]):
        qc, qs = quantise(x[which], fmt)
        codes, scales = codes.clone().view(t.int8).cpu(), scales.clone().cpu()
        back = t.zeros(R, hk, dim)
        r = 0
        for b, n in enumerate(rows):
            for i in range(n):
                pos = lens[b] - n + i
                if pos >= 0:
                    pg, o = int(c.table[b, pos // PAGE]), pos % PAGE
                    codes[pg, :, o] = qc[r].view(t.int8)
                    scales[pg, :, o] = qs[r]
                    back[r] = qc[r].float() * qs[r][:, None]
                r += 1
        want.append((codes, scales, back))
    serving.kvq_write(c.pool, c.batch, x[0].cuda(), x[1].cuda())
    k, v = serving.kvq_read(c.pool, c.batch, R, _types()[typ])
    for (codes, scales, back), gc, gs, gb in zip(want, (c.pool.k, c.pool.v), (c.pool.k_scale, c.pool.v_scale), (k, v)):
        assert t.equal(gc.view(t.int8).cpu(), codes)
        assert np.array_equal(gs.cpu().numpy(), scales.numpy(), equal_nan=True)
        assert np.array_equal(gb.float().cpu().numpy(), back.to(_types()[typ]).float().numpy(), equal_nan=True)


def test_write_takes_strided_and_unaligned_rows(gpu):
    t = _torch()
    from dotllm_b200 import serving
    for shift in (0, 1):  # shift 1: rows start off every 16-byte boundary
        a, b = Case("i8", 4, 128, [40, 70], [9, 30], seed=1), Case("i8", 4, 128, [40, 70], [9, 30], seed=1)
        flat = t.randn(39 * 3 * 512 + 8, device="cuda").half()
        qkv = flat[shift:shift + 39 * 3 * 512].view(39, 3, 4, 128)
        serving.kvq_write(a.pool, a.batch, qkv[:, 1], qkv[:, 2])
        serving.kvq_write(b.pool, b.batch, qkv[:, 1].clone(), qkv[:, 2].clone())
        assert t.equal(a.pool.k, b.pool.k) and t.equal(a.pool.v, b.pool.v)
        assert t.equal(a.pool.k_scale.nan_to_num(-1), b.pool.k_scale.nan_to_num(-1))


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("hk,g,dim,lens,rows,prefix", [
    (2, 4, 64, [1], [1], 0),                       # the first token of a sequence
    (2, 4, 64, [70], [1], 130),
    (1, 1, 96, [64, 65, 1, 300], [1, 1, 1, 1], 64),
    (2, 8, 128, [200, 33], [3, 5], 65),            # drafts, 24 and 40 rows per kv head
    (3, 1, 256, [63, 129, 5], [2, 1, 5], 1),
    (1, 16, 128, [10, 700], [1, 1], 0),
    (4, 3, 96, [300, 7], [70, 7], 100),            # a prompt chunk: many rows of one sequence
    (1, 2, 64, [5, 9, 1000], [0, 9, 2], 257)])     # a sequence without rows
def test_attention(gpu, typ, fmt, hk, g, dim, lens, rows, prefix):
    c = Case(fmt, hk, dim, lens, rows, prefix=prefix, seed=11)
    check_attention(c, rand_q(sum(rows), hk * g, dim, typ, 7), typ)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 7, 64, 150])
@pytest.mark.parametrize("dim", [64, 256])
def test_attention_window_and_softcap(gpu, typ, window, dim):
    """A window that cuts the prefix for some rows, and one that hides it from all."""
    c = Case("i8", 2, dim, [3, 140, 260], [3, 4, 1], prefix=90, seed=2)
    check_attention(c, rand_q(8, 4, dim, typ, 9, 4.0), typ, window=window, softcap=5.0)
    check_attention(c, rand_q(8, 4, dim, typ, 9), typ, window=window)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("batch", [40, 150])
def test_attention_many_rows_on_one_prefix(gpu, batch, dim):
    """Hundreds of rows per kv head over one prefix (the wide tiles), ragged rows and lengths."""
    rows = [1 + i % 4 for i in range(batch)]
    lens = [rows[i] + (i * 29) % 130 for i in range(batch)]
    for fmt, typ, window in (("i8", "bf16", 0), ("e4m3", "f16", 0), ("i8", "f32", 0), ("i8", "f16", 300)):
        c = Case(fmt, 1, dim, lens, rows, prefix=449, seed=4)
        check_attention(c, rand_q(sum(rows), 4, dim, typ, 3), typ, window=window)


def test_attention_rows_that_see_nothing(gpu):
    """More rows than positions and no prefix, an empty sequence with a row, and an empty batch."""
    t = _torch()
    c = Case("i8", 2, 64, [2, 0, 70], [4, 1, 2], seed=6)
    out, lse = check_attention(c, rand_q(7, 4, 64, "f16"), "f16")
    assert t.isinf(lse[:2]).all() and (out[:2] == 0).all() and t.isinf(lse[4]).all()
    c = Case("i8", 2, 64, [0, 0], [0, 0], seed=6)
    out, lse = c.attend(rand_q(0, 4, 64, "f16"))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_attention_skips_pages_outside_the_pool(gpu):
    """A page id outside the pool is not followed: its positions are not seen, everything else is."""
    t = _torch()
    c = Case("i8", 2, 128, [300, 200], [2, 1], prefix=100, seed=8)
    for bad in (-1, c.pool.n_pages, 2 ** 31 - 1):
        table = c.batch.pages.clone()
        table[0, 1] = bad
        from dotllm_b200 import serving
        keep, c.batch = c.batch, serving.KvqBatch(c.batch.row_start, c.batch.seq_len, table, 2)
        check_attention(c, rand_q(3, 4, 128, "f16"), "f16", hidden=[(0, j) for j in range(64, 128)])
        c.batch = keep
    # a list shorter than the sequence: positions beyond it are not seen
    from dotllm_b200 import serving
    c.batch = serving.KvqBatch(c.batch.row_start, c.batch.seq_len, c.batch.pages[:, :3].contiguous(), 2)
    check_attention(c, rand_q(3, 4, 128, "f16"), "f16", hidden=[(0, j) for j in range(192, 300)] + [(1, j) for j in range(192, 200)])


@pytest.mark.parametrize("typ,scale", [("f32", 1.0), ("bf16", 1e-6), ("f32", 1e-20), ("f16", 6e-5), ("bf16", 30.0), ("f32", 300.0)])
def test_attention_ranges(gpu, typ, scale):
    """Tiny and huge queries (a softmax that is flat, or takes one position), values over ten binary orders."""
    c = Case("e4m3", 2, 128, [200, 64], [2, 1], prefix=70, seed=9, v_spread=10.0)
    check_attention(c, rand_q(3, 8, 128, typ, 1, scale), typ)


def test_attention_nan_stays_with_the_rows_that_see_it(gpu):
    """A position whose scale is NaN makes the outputs of rows that see it NaN, and no others."""
    t = _torch()
    for dim in (64, 128, 256):
        c = Case("i8", 2, dim, [130, 90], [3, 2], prefix=70, seed=10)
        q = rand_q(5, 4, dim, "f16")
        clean, _ = c.attend(q)
        pos = 128  # seen by the last two rows of sequence 0
        c.pool.v_scale[int(c.table[0, 2]), 1, pos % PAGE] = float("nan")
        out, _ = c.attend(q)
        assert t.isnan(out[1:3, 2:]).all()
        assert t.equal(out[:1], clean[:1]) and t.equal(out[3:], clean[3:]) and t.equal(out[1:3, :2], clean[1:3, :2])


def test_attention_strided_queries_and_single_kv_page_reuse(gpu):
    """q as a slice of a fused projection; two sequences that list the same page."""
    t = _torch()
    c = Case("e4m3", 2, 64, [128, 128], [1, 2], prefix=10, seed=12)
    qkv = t.randn(3, 8 + 4, 64, device="cuda").half()
    out, lse = c.attend(qkv[:, 2:10])
    want, wlse = c.attend(qkv[:, 2:10].contiguous())
    assert t.equal(out, want) and t.equal(lse, wlse)
    odd = t.randn(3 * 8 * 64 + 1, device="cuda").half()[1:].view(3, 8, 64)
    assert t.equal(c.attend(odd)[0], c.attend(odd.clone())[0])
    from dotllm_b200 import serving
    table = c.batch.pages.clone()
    table[1, 0] = table[0, 0]
    c.kv[0][1][:64], c.kv[1][1][:64] = c.kv[0][0][:64], c.kv[1][0][:64]
    c.batch = serving.KvqBatch(c.batch.row_start, c.batch.seq_len, table, 2)
    check_attention(c, rand_q(3, 8, 64, "f16"), "f16")


def test_attention_same_result_every_time(gpu):
    t = _torch()
    c = Case("i8", 2, 128, [900, 65, 1300], [2, 1, 3], prefix=700, seed=13)
    q = rand_q(6, 8, 128, "bf16")
    first = c.attend(q)
    for _ in range(5):
        again = c.attend(q)
        assert t.equal(first[0], again[0]) and t.equal(first[1], again[1])


def test_offsets_beyond_32_bits(gpu):
    """Pages whose byte offset in the pool exceeds 2^32 (and whose element index exceeds 2^31)."""
    t = _torch()
    from dotllm_b200 import serving
    hk, dim, n_pages = 8, 128, 70000  # 4.6 GB of codes each for K and V
    pool = serving.KvqPool(t.empty(n_pages, hk, PAGE, dim, dtype=t.int8, device="cuda"),
                           t.empty(n_pages, hk, PAGE, dim, dtype=t.int8, device="cuda"),
                           t.empty(n_pages, hk, PAGE, device="cuda"), t.empty(n_pages, hk, PAGE, device="cuda"))
    low = Case("i8", hk, dim, [100, 70], [100, 70], prefix=64, seed=14)
    ids = {int(p): i for i, p in enumerate([*low.prefix_ids, *low.table[0, :2], *low.table[1, :2]])}
    high = t.tensor([[n_pages - 1 - ids[int(p)] if p >= 0 else -1 for p in row] for row in low.table], dtype=t.int32).cuda()
    pre = t.tensor([n_pages - 1 - ids[int(low.prefix_ids[0])]], dtype=t.int32).cuda()
    k, v = serving.kvq_read(low.pool, low.batch, 170)
    batch = serving.KvqBatch(low.batch.row_start, low.batch.seq_len, high, 100)
    serving.kvq_write(pool, batch, k, v)
    one = t.tensor([0, 64], dtype=t.int32).cuda()
    pb_low = serving.KvqBatch(one, one[1:].contiguous(), low.prefix_pages.view(1, 1), 64)
    pb_high = serving.KvqBatch(one, one[1:].contiguous(), pre.view(1, 1), 64)
    serving.kvq_write(pool, pb_high, *serving.kvq_read(low.pool, pb_low, 64))
    back = serving.kvq_read(pool, batch, 170)
    again = Case("i8", hk, dim, [100, 70], [100, 70], prefix=64, seed=14)  # the same through low pages
    serving.kvq_write(again.pool, again.batch, k, v)
    serving.kvq_write(again.pool, pb_low, *serving.kvq_read(low.pool, pb_low, 64))
    for x, y in zip(back, serving.kvq_read(again.pool, again.batch, 170)):
        assert t.equal(x, y)
    q = rand_q(170, 8, dim, "f16")
    a = serving.kvq_attention(pool, batch, q, prefix_pages=pre, prefix_len=64)
    b = serving.kvq_attention(again.pool, again.batch, q, prefix_pages=again.prefix_pages, prefix_len=64)
    assert t.equal(a, b)


def test_streams_and_graph_capture(gpu):
    """Calls order with other work of the current stream, and replay from a CUDA graph with new lengths."""
    t = _torch()
    from dotllm_b200 import serving
    c = Case("i8", 2, 128, [200, 100], [2, 1], prefix=70, seed=15)
    q = rand_q(3, 8, 128, "f16")
    x = [t.randn(3, 2, 128, device="cuda").half() for _ in range(2)]
    p = t.softmax(t.randn(2, 4, 1000, device="cuda"), -1)
    dq = t.softmax(t.randn(2, 3, 1000, device="cuda"), -1)
    draft = t.randint(0, 1000, (2, 3), device="cuda", dtype=t.int32)
    u = t.rand(2, 4, device="cuda")

    def step(q, x, u):
        serving.kvq_write(c.pool, c.batch, *x)
        return (*serving.kvq_read(c.pool, c.batch, 3, t.float16), *c.attend(q), *serving.verify_draft(p, dq, draft, u))

    want = [o.clone() for o in step(q, x, u)]
    t.cuda.synchronize()
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        late = [t.zeros_like(q), [t.zeros_like(y) for y in x], t.zeros_like(u)]
        t.cuda._sleep(20_000_000)  # the inputs arrive late on this stream
        late[0].copy_(q)
        late[1][0].copy_(x[0])
        late[1][1].copy_(x[1])
        late[2].copy_(u)
        got = step(*late)
    side.synchronize()
    assert all(t.equal(a, b) for a, b in zip(want, got))
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        got = step(q, x, u)
    q.copy_(q.flip(0))
    c.batch.seq_len.copy_(t.tensor([190, 30], dtype=t.int32))
    want = [o.clone() for o in step(q, x, u)]
    for o in got:
        o.zero_()
    graph.replay()
    t.cuda.synchronize()
    assert all(t.equal(a, b) for a, b in zip(want, got))


# ------------------------------------------------------------------ verification
def verify_reference(p, q, draft, u, n_draft):
    """The definition in Python integers."""
    f = np.float32
    B, k1, V = p.shape
    k = k1 - 1
    tokens, accepted = np.full((B, k1), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        n = int(n_draft[b])
        a = 0
        while a < n:
            x = int(draft[b, a])
            if not 0 <= x < V:
                break
            qx = q[b, a, x] if q is not None else f(1)
            if not f(u[b, a]) * f(qx) < p[b, a, x]:
                break
            a += 1
        w = p[b, a].astype(f)
        if a < n:
            less = q[b, a] if q is not None else np.zeros(V, f)
            if q is None and 0 <= draft[b, a] < V:
                less[draft[b, a]] = 1
            w = (w - less).astype(f)

        def ints(w):
            w = np.clip(np.where(np.isnan(w), f(0), w), f(0), f(1)).astype(f)
            return [int(x) for x in np.floor(w.astype(np.float64) * 2.0 ** 40)]
        W = ints(w)
        if sum(W) == 0:
            W = ints(p[b, a])
        T = sum(W)
        t = int(np.floor(float(u[b, k]) * 2.0 ** 24)) * T >> 24
        pick, run = 0, 0
        for j, x in enumerate(W):
            run += x
            if run > t:
                pick = j
                break
        tokens[b, :a] = draft[b, :a]
        tokens[b, a] = pick
        accepted[b] = a
    return tokens, accepted


def check_verify(p, q, draft, u, n_draft=None):
    t = _torch()
    from dotllm_b200 import serving
    B, k1, V = p.shape
    n = np.full(B, k1 - 1) if n_draft is None else n_draft
    tok, acc = serving.verify_draft(t.from_numpy(p).cuda(), None if q is None else t.from_numpy(q).cuda(),
                                    t.from_numpy(draft.astype(np.int32)).cuda(), t.from_numpy(u).cuda(),
                                    None if n_draft is None else t.from_numpy(n.astype(np.int32)).cuda())
    want, wacc = verify_reference(p, q, draft, u, n)
    assert np.array_equal(acc.cpu().numpy(), wacc)
    assert np.array_equal(tok.cpu().numpy(), want)
    return want, wacc


def probs(rng, *shape, sharp=2.0):
    x = rng.standard_normal(shape) * sharp
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 31, 33, 127, 128, 1000, 1025, 4099, 50257])
@pytest.mark.parametrize("with_q", [True, False])
def test_verify(gpu, V, with_q):
    rng = np.random.default_rng(V + with_q)
    B, k = (12, 5) if V < 10000 else (4, 3)
    p, q = probs(rng, B, k + 1, V), probs(rng, B, k, V)
    q = (0.3 * q + 0.7 * p[:, :k]).astype(np.float32)
    draft = np.array([[rng.choice(V, p=q[b, i].astype(np.float64) / q[b, i].sum(dtype=np.float64)) for i in range(k)] for b in range(B)])
    u = rng.random((B, k + 1), dtype=np.float32)
    u[0, k], u[1, k] = 0.0, np.float32(1) - np.float32(2.0 ** -24)
    _, acc = check_verify(p, q if with_q else None, draft, u)
    check_verify(p, q if with_q else None, draft, u, rng.integers(0, k + 1, B))


def test_verify_extremes(gpu):
    """Everything refused, everything accepted, p equal to q, rows of zeros, NaN and infinities, tokens
    outside the vocabulary, no drafts at all, one-hot rows, a full 64 drafts."""
    rng = np.random.default_rng(0)
    f = np.float32
    B, k, V = 10, 4, 300
    p, q = probs(rng, B, k + 1, V), probs(rng, B, k, V)
    draft = rng.integers(0, V, (B, k))
    u = rng.random((B, k + 1), dtype=np.float32)
    u[0, :k] = 0                                  # all accepted
    q[1] = p[1, :k]
    u[1, 0] = f(1) - f(2.0 ** -24)
    draft[2, 0], draft[3, 1] = -1, V              # outside the vocabulary
    u[3] = 0
    p[4, 0] = 0                                   # nothing in p: token 0
    p[5, 0] = 0
    p[5, 0, 7] = 1                                # one-hot target
    p[6, 0, 5], p[6, 0, 9], q[6, 0, 11] = np.nan, np.inf, np.nan
    q[7] = 2.0                                    # residual weighs nothing: p's own weights
    p[8, 0], q[8, 0] = f(2.0 ** -41), 0           # every weight below one unit
    check_verify(p, q, draft, u)
    check_verify(p, None, draft, u)
    check_verify(p[:, :1].copy(), np.zeros((B, 0, V), f), np.zeros((B, 0), np.int32), u[:, k:].copy())
    p, q = probs(rng, 3, 65, 50, sharp=0.3), probs(rng, 3, 64, 50, sharp=0.3)
    draft = rng.integers(0, 50, (3, 64))
    u = np.zeros((3, 65), f)
    u[1, 40] = u[2, 63] = f(0.99999)
    p[1, 40, draft[1, 40]] = p[2, 63, draft[2, 63]] = 0
    _, acc = check_verify(p, q, draft, u)
    assert acc.tolist() == [64, 40, 63]


def test_verify_keeps_the_targets_distribution(gpu):
    """Over many draws the emitted token follows the target's probabilities, whatever drafted it."""
    t = _torch()
    from dotllm_b200 import serving
    rng = np.random.default_rng(1)
    N, V = 200000, 6
    p1, q1 = probs(rng, V, sharp=1.0), probs(rng, V, sharp=1.0)
    draft = rng.choice(V, size=(N, 1), p=q1.astype(np.float64) / q1.sum(dtype=np.float64)).astype(np.int32)
    p = t.from_numpy(np.stack([p1, p1])).cuda()[None].expand(N, 2, V).contiguous()
    q = t.from_numpy(q1).cuda()[None, None].expand(N, 1, V).contiguous()
    tok, _ = serving.verify_draft(p, q, t.from_numpy(draft).cuda(), t.rand(N, 2, device="cuda", generator=t.Generator("cuda").manual_seed(2)))
    got = np.bincount(tok[:, 0].cpu().numpy(), minlength=V) / N
    sigma = np.sqrt(p1 * (1 - p1) / N)
    assert (np.abs(got - p1) < 5 * sigma + 1e-6).all(), (got, p1)


def test_verify_strided_rows(gpu):
    t = _torch()
    from dotllm_b200 import serving
    rng = np.random.default_rng(3)
    p, q = t.from_numpy(probs(rng, 6, 4, 777)).cuda(), t.from_numpy(probs(rng, 6, 3, 777)).cuda()
    wide = t.zeros(6, 4, 800, device="cuda")
    wide[..., :777] = p
    draft, u = t.randint(0, 777, (6, 3), device="cuda", dtype=t.int32), t.rand(6, 4, device="cuda")
    a, b = serving.verify_draft(p, q, draft, u), serving.verify_draft(wide[..., :777], q, draft, u)
    assert t.equal(a[0], b[0]) and t.equal(a[1], b[1])


# ------------------------------------------------------------------ refusals that need tensors
def test_refusals(gpu):
    t = _torch()
    from dotllm_b200 import serving
    c = Case("i8", 2, 64, [10, 20], [1, 1], seed=1)
    x = t.randn(2, 2, 64, device="cuda")
    q = t.randn(2, 4, 64, device="cuda")
    for bad in (lambda: serving.kvq_write(c.pool, c.batch, x.double(), x.double()),
                lambda: serving.kvq_write(c.pool, c.batch, x, x.half()),
                lambda: serving.kvq_write(c.pool, c.batch, x[:, :1], x[:, :1]),
                lambda: serving.kvq_write(c.pool, c.batch, x.transpose(0, 1).contiguous().transpose(0, 1), x),
                lambda: serving.kvq_write(c.pool, c.batch, x.cpu(), x.cpu()),
                lambda: serving.kvq_read(c.pool, c.batch, 2, t.int8),
                lambda: serving.kvq_read(c.pool, c.batch, -1),
                lambda: c.attend(q[..., :32]),
                lambda: c.attend(q.to(t.int8)),
                lambda: serving.kvq_attention(c.pool, c.batch, q, prefix_len=5),
                lambda: serving.kvq_attention(c.pool, c.batch, q, prefix_pages=t.zeros(1, dtype=t.int32, device="cuda"), prefix_len=65),
                lambda: serving.kvq_attention(c.pool, c.batch, q, prefix_pages=t.zeros(2, device="cuda"), prefix_len=65),
                lambda: serving.KvqPool(c.pool.k, c.pool.v[:1], c.pool.k_scale, c.pool.v_scale),
                lambda: serving.KvqPool(c.pool.k.float(), c.pool.v.float(), c.pool.k_scale, c.pool.v_scale),
                lambda: serving.KvqBatch(c.batch.row_start[:2], c.batch.seq_len, c.batch.pages, 1),
                lambda: serving.KvqBatch(c.batch.row_start.long(), c.batch.seq_len, c.batch.pages, 1),
                lambda: serving.verify_draft(t.rand(2, 3, 9, device="cuda"), None, t.zeros(2, 3, dtype=t.int32, device="cuda"),
                                             t.rand(2, 3, device="cuda")),
                lambda: serving.verify_draft(t.rand(2, 3, 9, device="cuda"), t.rand(2, 2, 8, device="cuda"),
                                             t.zeros(2, 2, dtype=t.int32, device="cuda"), t.rand(2, 3, device="cuda")),
                lambda: serving.verify_draft(t.rand(2, 3, 9, device="cuda").half(), None, t.zeros(2, 2, dtype=t.int32, device="cuda"),
                                             t.rand(2, 3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    from dotllm_b200.native import CudaBackendError
    for bad in (lambda: c.attend(t.randn(2, 3, 64, device="cuda")),            # heads not a multiple of heads_kv
                lambda: c.attend(q, window=-1), lambda: c.attend(q, softcap=-1.0), lambda: c.attend(q, softcap=float("nan")),
                lambda: c.attend(q, scale=float("inf")),
                lambda: serving.KvqPool.empty(3, 2, 80) and serving.kvq_read(serving.KvqPool.empty(3, 2, 80), c.batch, 2),
                lambda: serving.verify_draft(t.rand(1, 70, 9, device="cuda"), None, t.zeros(1, 69, dtype=t.int32, device="cuda"),
                                             t.rand(1, 70, device="cuda"))):
        with pytest.raises(CudaBackendError):
            bad()
