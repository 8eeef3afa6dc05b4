"""Shared-prefix attention where the values' scales or the softmax are far from even: value rows that are many binary
orders larger than the others at positions that a row does not see, or sees with next to no weight; an attention
sink whose own value is small; missing pages and NaN scales under the many-row kernel.

Every (row, head) is held to its own bar, from what that row sees alone.  With w_j its softmax weights,
X the largest sum |q_i k_i| scale, e = 2^-21 X what a score may be off by (fp32 sums in any order), N its positions:

* each output value: A = sum w_j |v_j| times (2 e + 2^-18 + W), W = 2^-11 for bf16 queries, whose weights are rounded to
  11 bits, 2^-21 else; N 2^-28 max w_j |v_j|_inf, since weights may end 2^-28 below a row's largest; half a unit
  in the last place of the output type (2^-8 of a value with 8 significant bits, 2^-11 with 11); the smallest steps of
  the types count as they are;
  Where one thread block adds up C positions one after another (check's `chain`), C 2^-26 A more: 16 positions
  an addition, of hi and of lo, each truncated at 2^-23 of the sum;
* the row in the norm: the weights' roundings are independent and v's signs random (or all alike), so they add W |out|,
  not W A; the output's roundings are even in half a unit, 2^-8 / sqrt(3) (bf16) |out| at most, or 2^-11 (fp16).
  Bars of 3e-3 (2^-8 / sqrt(3) + 2^-11 = 2.75e-3), 5.5e-4 and 2 e + 2^-17.
"""
import pytest

pytestmark = pytest.mark.gpu
PAGE = 64
TYPES = ["f32", "f16", "bf16"]
WEIGHT = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -11}
ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -140, "f16": 2.0 ** -25, "bf16": 2.0 ** -130}
NORM = {"f32": 0.0, "f16": 5.5e-4, "bf16": 3e-3}


class Held:
    """A pool whose unused slots hold garbage and the values that its codes stand for.  parts: K and V [n, hk, dim] of the
    prefix, then of each sequence."""

    def __init__(self, fmt, parts, rows, seed=0):
        import torch
        from dotllm_b200 import serving
        g = torch.Generator("cuda").manual_seed(seed)
        (hk, dim), lens = parts[0][0].shape[1:], [p[0].shape[0] for p in parts]
        need = [-(-n // PAGE) for n in lens]
        ids = torch.randperm(sum(need) + 2, device="cuda", generator=g).int()
        lists, at = [], 0
        for n in need:
            lists.append(ids[at:at + n].contiguous())
            at += n
        self.table = torch.full((len(rows), max(need[1:] + [1]) + 1), -1, dtype=torch.int32, device="cuda")
        for b, p in enumerate(lists[1:]):
            self.table[b, :len(p)] = p
        top = 127.0 if fmt == "i8" else 448.0
        self.values, pool = [], []
        for which in range(2):
            codes = torch.full((len(ids), hk, PAGE, dim), -1, dtype=torch.int8, device="cuda")
            scales = torch.full((len(ids), hk, PAGE), float("nan"), device="cuda")
            held = []
            for x, pages in zip((p[which] for p in parts), lists):
                s = x.abs().amax(-1) / top
                c = x / torch.where(s > 0, s, 1.0)[..., None]
                c = torch.round(c).clamp(-127, 127).to(torch.int8) if fmt == "i8" else c.clamp(-448, 448).to(torch.float8_e4m3fn)
                j = torch.arange(x.shape[0], device="cuda")
                if len(j):
                    codes[pages[j // PAGE].long(), :, j % PAGE] = c.view(torch.int8)
                    scales[pages[j // PAGE].long(), :, j % PAGE] = s
                held.append(c.double() * s.double()[..., None])
            self.values.append(held)
            pool += [codes.view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn), scales]
        self.pool = serving.KvqPool(pool[0], pool[2], pool[1], pool[3])
        self.rows, self.lens, self.prefix, self.prefix_pages, self.lists = rows, lens[1:], lens[0], lists[0], lists
        self.row_start = torch.tensor([0] + rows, device="cuda").cumsum(0).int()
        self.seq_len = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def attend(self, q, table=None, prefix_pages=None, **kw):
        from dotllm_b200 import serving
        batch = serving.KvqBatch(self.row_start, self.seq_len, self.table if table is None else table, max(self.rows))
        return serving.kvq_attention(self.pool, batch, q, prefix_len=self.prefix, return_lse=True,
                                     prefix_pages=self.prefix_pages if prefix_pages is None else prefix_pages, **kw)

    def check(self, q, typ, got, window=0, softcap=0.0, hidden=None, only=None, chain=0):
        """got = (out, lse) against 64 bits; hidden(b): positions of the whole that sequence b does not see; only: the
        rows (their numbers in a sequence) that are checked; chain: positions added up one after another."""
        import torch
        out, lse = got
        R, H, D = q.shape
        hk = self.pool.heads_kv
        G, r = H // hk, 0
        for b, n in enumerate(self.rows):
            k = torch.cat([self.values[0][0], self.values[0][1 + b]]).transpose(0, 1)
            v = torch.cat([self.values[1][0], self.values[1][1 + b]]).transpose(0, 1)
            T = self.prefix + self.lens[b]

            def rows_of(x):
                return x[r:r + n].double().reshape(n, hk, G, -1).permute(1, 0, 2, 3).reshape(hk, n * G, -1)

            x = rows_of(q)
            s = x @ k.transpose(1, 2) * D ** -0.5
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            p = T - n + torch.arange(n, device="cuda").repeat_interleave(G)[:, None]
            j = torch.arange(T, device="cuda")[None]
            gone = (j > p) | (j <= p - (window or T + n))
            if hidden is not None:
                gone = gone | torch.isin(j, torch.as_tensor(hidden(b), device="cuda"))
            seen = ~gone[None]
            big = (x.abs() @ k.abs().transpose(1, 2) * D ** -0.5).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            s = s.masked_fill(~seen, float("-inf"))
            want_lse = torch.logsumexp(s, -1, keepdim=True)
            w = torch.where(torch.isinf(want_lse), 0.0, torch.exp(s - want_lse))
            v = torch.where(torch.isfinite(v), v, 0.0)  # (a position that is NaN is none that a checked row sees)
            want, A = w @ v, w @ v.abs()
            e = 2.0 ** -21 * big
            floor = T * 2.0 ** -28 * (w * v.abs().amax(-1)[:, None]).amax(-1, keepdim=True)
            bar = A * (2 * e + 2.0 ** -18 + chain * 2.0 ** -26 + WEIGHT[typ]) + floor + want.abs() * ROUND[typ] + LEAST[typ]
            a, al = rows_of(out), rows_of(lse[..., None])
            norm, err = want.norm(dim=-1, keepdim=True), (a - want).norm(dim=-1, keepdim=True)
            norm_bar = norm * (NORM[typ] or 2.0 ** -17) + chain * 2.0 ** -26 * A.norm(dim=-1, keepdim=True) + 2 * e * norm + floor * D ** 0.5 + LEAST[typ] * D ** 0.5
            pick = torch.ones(n, dtype=torch.bool, device="cuda")
            if only is not None:
                pick = torch.isin(torch.arange(n, device="cuda"), torch.tensor(list(only), device="cuda"))
            pick = pick.repeat_interleave(G)
            rel = (err / norm.clamp(min=1e-300))[:, pick]
            assert torch.isfinite(a[:, pick]).all()
            assert ((a - want).abs() <= bar)[:, pick].all(), (b, float(rel.max()))
            assert (err <= norm_bar)[:, pick].all(), (b, float(rel.max()))
            known = ~torch.isinf(want_lse)
            assert (torch.isinf(al) == ~known)[:, pick].all()
            far = (al - want_lse).abs() > e + 2.0 ** -20 * (1 + want_lse.abs())
            assert not (far & known)[:, pick].any()
            r += n


def noise(seed, *shape):
    import torch
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def queries(seed, typ, *shape, scale=1.0):
    import torch
    return (noise(seed, *shape) * scale).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[typ])


def random_parts(seed, hk, dim, *lens):
    return [(noise(seed + 2 * i, n, hk, dim), noise(seed + 2 * i + 1, n, hk, dim)) for i, n in enumerate(lens)]


# group 2: few rows per kv head; group 20: 60 and more, the many-row kernel (for 16-bit queries)
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (96, "e4m3"), (128, "i8"), (256, "e4m3")])
@pytest.mark.parametrize("group", [2, 20])
def test_large_value_of_a_later_row(gpu, typ, dim, fmt, group):
    """The last drafted row's own value is 2^k times the others': the earlier rows, which do not see it, keep their precision."""
    for k in (8, 12, 16, 20, 40):
        parts = random_parts(k, 2, dim, 70, 60, 9)
        parts[1][1][-1] *= 2.0 ** k
        c = Held(fmt, parts, [3, 2])
        q = queries(1, typ, 5, 2 * group, dim)
        c.check(q, typ, c.attend(q), only=(0, 1) if typ == "f16" else None)  # (2^40 is beyond fp16)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", [(64, "e4m3"), (96, "i8"), (128, "e4m3"), (256, "i8")])
@pytest.mark.parametrize("group", [2, 20])
def test_large_value_outside_the_window(gpu, typ, dim, fmt, group):
    """The same at positions that the window hides, before (in the prefix's page that is still read) and in own pages."""
    for k in (8, 12, 16, 20, 40):
        parts = random_parts(k, 2, dim, 150, 100)
        parts[0][1][:120] *= 2.0 ** k
        parts[0][1][120:] *= 2.0 ** -3
        c = Held(fmt, parts, [3])
        q = queries(2, typ, 3, 2 * group, dim)
        c.check(q, typ, c.attend(q, window=125), window=125)  # the first row sees from position 123 on
        parts = random_parts(k, 2, dim, 0, 130)
        parts[1][1][:70] *= 2.0 ** k
        c = Held(fmt, parts, [3])
        c.check(q, typ, c.attend(q, window=50), window=50)  # from position 78 on


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (96, "e4m3"), (128, "i8"), (256, "e4m3")])
@pytest.mark.parametrize("group", [2, 20])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_large_value_with_next_to_no_weight(gpu, typ, dim, fmt, group, softcap):
    """A position that every row sees with a weight of 2^-50 or less, its value 2^20 times the others': what it adds is
    far below the others' rounding, first or last in the order of pages, and they keep theirs."""
    for at in (0, 199):
        parts = random_parts(at, 2, dim, 200, 40)
        for part in parts:
            part[0][..., 0] = 0.0
        parts[0][0][at] = 0.0
        parts[0][0][at, :, 0] = -40.0 * dim ** 0.5 / 4.0  # a score of -40, -30 tanh(4 / 3) under the cap
        parts[0][1][at] *= 2.0 ** 12 if softcap else 2.0 ** 20
        c = Held(fmt, parts, [4])
        q = queries(3, typ, 4, 2 * group, dim)
        q[..., 0] = 4.0
        c.check(q, typ, c.attend(q, softcap=softcap), softcap=softcap)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (96, "e4m3"), (128, "i8"), (256, "e4m3")])
@pytest.mark.parametrize("group", [2, 20])
def test_value_scales_of_every_size(gpu, typ, dim, fmt, group):
    """All values tiny, all huge, and orders that change from page to page, up and down."""
    sizes = [0, -8, 3] if typ == "f16" else [0, -90, 100]
    for k in sizes:
        parts = random_parts(k + 100, 2, dim, 130, 70)
        for _, v in parts:
            v *= 2.0 ** k
        c = Held(fmt, parts, [3])
        q = queries(4, typ, 3, 2 * group, dim)
        c.check(q, typ, c.attend(q))
    steps = [5, -6, 0, -9] if typ == "f16" else [40, -40, 0, -60]
    for order in (steps, steps[::-1]):
        parts = random_parts(7, 2, dim, 256, 70)
        for i, k in enumerate(order):
            parts[0][1][64 * i:64 * (i + 1)] *= 2.0 ** k
        c = Held(fmt, parts, [3])
        q = queries(5, typ, 3, 2 * group, dim)
        c.check(q, typ, c.attend(q))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("group", [2, 20])
def test_values_of_zero_under_a_large_score(gpu, typ, group):
    """A position that takes nearly all the weight and whose value is zero, by scores of up to 100: what is left of the
    others is still right to a row's own precision."""
    import torch
    for score in (10.0, 40.0, 80.0):
        parts = random_parts(11, 2, 128, 300, 30)
        for part in parts:
            part[0][..., 0] = 0.0
        parts[0][0][100] = 0.0
        parts[0][0][100, :, 0] = score * 128 ** 0.5 / 4.0
        parts[0][1][100] = 0.0
        c = Held("i8", parts, [3])
        q = queries(6, typ, 3, 2 * group, 128)
        q[..., 0] = 4.0
        out, lse = c.attend(q)
        c.check(q, typ, (out, lse))
        if typ != "f16":
            assert bool((out != 0).any()) and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (128, "e4m3"), (256, "i8")])
@pytest.mark.parametrize("group", [2, 20])
def test_attention_sink(gpu, typ, dim, fmt, group):
    """The first position takes most of the weight and has a small value, as a model's first token often does: the output
    is made of the many small weights."""
    for gap in (8.0, 10.0, 11.0, 13.0):
        parts = random_parts(12, 2, dim, 4096, 70)
        for part in parts:
            part[0][..., 0] = 0.0
        parts[0][0][0] = 0.0
        parts[0][0][0, :, 0] = gap * dim ** 0.5 / 4.0
        parts[0][1][0] *= 0.01
        c = Held(fmt, parts, [3])
        q = queries(7, typ, 3, 2 * group, dim, scale=0.3)
        q[..., 0] = 4.0
        c.check(q, typ, c.attend(q))

@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_tail_of_small_weights(gpu, typ, dim):
    """A sink among 32768 positions that one thread block goes through (1024 rows of each of 32 kv heads, so nothing is cut
    along the positions): the others weigh 2^-17 of it each, a fifth of it together, and the values have a common part."""
    parts = random_parts(13, 32, dim, 32768, 3)
    for k, v in parts:
        k.zero_()
        v.mul_(0.1).add_(1.0 + noise(14, 1, 32, dim).abs())
    parts[0][0][0, :, 0] = 12.0 * dim ** 0.5 / 4.0
    parts[0][1][0] = noise(15, 32, dim)
    c = Held("i8", parts[:1] + parts[1:] * 64, [1] * 64)
    q = queries(8, typ, 64, 32 * 16, dim, scale=0.3)
    q[..., 0] = 4.0
    c.check(q, typ, c.attend(q), chain=32768)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("group", [2, 20])
def test_negative_scales(gpu, typ, group):
    """A code stands for code * scale whatever the scale's sign."""
    parts = random_parts(16, 2, 128, 300, 70)
    c = Held("i8", parts, [3])
    for which, scales in ((0, c.pool.k_scale), (1, c.pool.v_scale)):
        scales[:, :, 1::3] *= -1.0
        for n, held in enumerate(c.values[which]):
            held[[j for j in range(held.shape[0]) if j % PAGE % 3 == 1]] *= -1.0
    q = queries(9, typ, 3, 2 * group, 128)
    c.check(q, typ, c.attend(q))


# 3 rows a sequence: 6, 18 and 60 per kv head on own pages, twice that on the prefix -- either side of where the kernels change
GROUPS = [2, 6, 20]
DIMS = [(64, "e4m3"), (96, "i8"), (128, "e4m3"), (256, "i8")]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", DIMS)
@pytest.mark.parametrize("group", GROUPS)
def test_pages_outside_the_pool(gpu, typ, dim, fmt, group):
    """Ids outside the pool, in a sequence's list or the prefix's, first, in the middle and last: never followed, not seen."""
    c = Held(fmt, random_parts(17, 2, dim, 300, 330, 200), [3, 3])
    q = queries(10, typ, 6, 2 * group, dim)
    for bad in (-1, c.pool.n_pages, 2 ** 31 - 1):
        for own, pre in ((1, None), (None, 2), (0, 0), (5, 4), (None, 0)):
            table, prefix_pages = c.table.clone(), c.prefix_pages.clone()
            gone = []
            if pre is not None:
                prefix_pages[pre] = bad
                gone += list(range(64 * pre, min(300, 64 * pre + 64)))
            if own is not None:
                table[0, own] = bad
            mine = [] if own is None else list(range(300 + 64 * own, 300 + min(330, 64 * own + 64)))
            got = c.attend(q, table=table, prefix_pages=prefix_pages)
            c.check(q, typ, got, hidden=lambda b: gone + (mine if b == 0 else []))
    table[:], prefix_pages[:] = -1, -1  # nothing at all
    out, lse = c.attend(q, table=table, prefix_pages=prefix_pages)
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("dim,fmt", DIMS)
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_nan_scales_reach_the_rows_that_see_them(gpu, typ, dim, fmt, group, softcap):
    """A NaN scale of K or V makes the rows NaN that see it, of its kv head; the others are what they are without it.  At the
    last drafted position, one before, and in the prefix where the window shows it to the first row alone."""
    import torch
    for which in ("k_scale", "v_scale"):
        for at, seen, window in ((329, (2,), 0), (328, (1, 2), 0), (-40, (0,), 368)):
            c = Held(fmt, random_parts(18, 2, dim, 300, 330, 200), [3, 3])
            q = queries(11, typ, 6, 2 * group, dim)
            pages, j = (c.lists[1], at) if at >= 0 else (c.lists[0], 300 + at)
            getattr(c.pool, which)[int(pages[j // PAGE]), 1, j % PAGE] = float("nan")
            held = c.values[0 if which == "k_scale" else 1][1 if at >= 0 else 0]
            held[j, 1] = float("nan")
            if at < 0:  # (both sequences have the prefix: the second's rows see it in the window, too)
                seen_by = {0: seen, 1: (0, 1, 2)}
            else:
                seen_by = {0: seen, 1: ()}
            out, lse = c.attend(q, window=window, softcap=softcap)
            clear = torch.ones(6, dtype=torch.bool)
            for b in (0, 1):
                for i in seen_by[b]:
                    clear[3 * b + i] = False
                    assert bool(torch.isnan(out[3 * b + i, group:]).all())
            held[j, 1] = 0.0
            assert bool(torch.isfinite(out[:, :group]).all()) and bool(torch.isfinite(out[clear.cuda()]).all())
            if at >= 0:
                c.check(q, typ, (out, lse), window=window, softcap=softcap, only=[i for i in range(3) if i not in seen])
            else:
                c.rows, keep = [3], c.rows
                c.check(q[:3], typ, (out[:3], lse[:3]), window=window, softcap=softcap, only=(1, 2))
                c.rows = keep


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("dim,fmt", DIMS)
@pytest.mark.parametrize("group", [2, 20])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_key_scales_of_every_size(gpu, typ, dim, fmt, group, softcap):
    """Keys tiny or huge and queries the inverse: the scores are ordinary, whatever the order of their factors."""
    for k in (-90, 110):
        parts = random_parts(k + 200, 2, dim, 130, 70)
        for key, _ in parts:
            key *= 2.0 ** k
        c = Held(fmt, parts, [3])
        q = queries(12, typ, 3, 2 * group, dim, scale=2.0 ** -k)
        c.check(q, typ, c.attend(q, softcap=softcap), softcap=softcap)


@pytest.mark.parametrize("dim,fmt", DIMS)
@pytest.mark.parametrize("group", [2, 20])
def test_subnormal_fp16_queries(gpu, dim, fmt, group):
    """fp16 queries below the smallest normal number, over keys that make ordinary scores of them."""
    parts = random_parts(19, 2, dim, 130, 70)
    for key, _ in parts:
        key *= 2.0 ** 17
    c = Held(fmt, parts, [3])
    q = queries(13, "f16", 3, 2 * group, dim, scale=2.0 ** -17)
    c.check(q, "f16", c.attend(q))
    c.check(q, "f16", c.attend(q, window=90), window=90)


@pytest.mark.parametrize("dim,fmt", [(64, "i8"), (96, "e4m3"), (128, "i8"), (256, "e4m3")])
@pytest.mark.parametrize("group,rows,prefix,own", [(2, [7] * 25, 2148, 17), (4, [100], 4000, 300), (1, [1], 0, 1900), (8, [1] * 3, 6239, 121)])
def test_fp32_sums_keep_32_bits(gpu, dim, fmt, group, rows, prefix, own):
    """fp32 queries: no further from 64 bits, in the norm of all rows, than torch operations in 32 bits are, but for 2^-20.  That is 2^-21
    for sums that the tensor core truncates (half a unit, 2^-24, an addition, eight additions before one that rounds), 2^-22 for
    the exponential and 2^-22 for queries and weights of 22 bits."""
    import torch
    hk = 4
    parts = random_parts(20, hk, dim, prefix, *[own] * len(rows))
    c = Held(fmt, parts, rows)
    q = queries(14, "f32", sum(rows), hk * group, dim)
    out = c.attend(q)[0]
    far, plain, size, r = 0.0, 0.0, 0.0, 0
    for b, n in enumerate(rows):
        T = prefix + own
        p = T - n + torch.arange(n, device="cuda").repeat_interleave(group)[:, None]
        gone = torch.arange(T, device="cuda")[None] > p

        def rows_of(x):
            return x[r:r + n].reshape(n, hk, group, dim).permute(1, 0, 2, 3).reshape(hk, n * group, dim)

        def attend(t):
            k, v = (torch.cat([x[0], x[1 + b]]).transpose(0, 1).to(t) for x in c.values)
            s = (rows_of(q).to(t) @ k.transpose(1, 2) * dim ** -0.5).masked_fill(gone, float("-inf"))
            w = torch.exp(s - s.amax(-1, keepdim=True))
            return (w @ v / w.sum(-1, keepdim=True)).double()

        want = attend(torch.float64)
        far += float((rows_of(out).double() - want).square().sum())
        plain += float((attend(torch.float32) - want).square().sum())
        size += float(want.square().sum())
        r += n
    assert (far / size) ** 0.5 <= (plain / size) ** 0.5 + 2.0 ** -20, ((far / size) ** 0.5, (plain / size) ** 0.5)
