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
