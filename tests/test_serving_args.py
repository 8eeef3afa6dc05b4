"""Argument checks of the serving operators' C entry points: refused before anything touches a device
(no GPU needed; nothing is launched)."""
import ctypes as C
import subprocess

import pytest

from dotllm_b200 import native

INVALID, UNSUPPORTED = -1, -2
P = 1 << 12  # a non-null, aligned address that is never followed


def pool(**kw):
    d = dict(format=0, head_dim=64, heads_kv=2, n_pages=4, k=P, v=P, k_scale=P, v_scale=P)
    d.update(kw)
    return native.KvqPool(**d)


def batch(**kw):
    d = dict(batch=1, rows=1, max_rows=1, max_pages=1, row_start=P, seq_len=P, pages=P)
    d.update(kw)
    return native.KvqBatch(**d)


def attn(**kw):
    d = dict(heads=4, type=1, prefix_len=0, window=0, scale=0.125, softcap=0.0, prefix_pages=None)
    d.update(kw)
    return native.KvqAttn(**d)


def message():
    return native.lib().llmdot_cuda_last_error().decode()


BAD_POOLS = [(dict(format=2), INVALID), (dict(head_dim=80), UNSUPPORTED), (dict(heads_kv=0), INVALID), (dict(n_pages=-1), INVALID),
             (dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(k=P + 8), INVALID), (dict(k_scale=P + 2), INVALID)]
BAD_BATCHES = [dict(batch=-1), dict(rows=-1), dict(max_rows=-1), dict(max_pages=-1), dict(max_pages=1 << 25), dict(row_start=None),
               dict(seq_len=None), dict(pages=None), dict(batch=0)]


def test_pool_and_batch_refusals():
    L = native.lib()
    need = C.c_size_t()
    calls = [lambda p, b: L.llmdot_cuda_kvq_write(p, b, P, P, 1, 128, 128, None),
             lambda p, b: L.llmdot_cuda_kvq_read(p, b, P, P, 1, 128, 128, None),
             lambda p, b: L.llmdot_cuda_kvq_attention_workspace(p, b, attn(), need),
             lambda p, b: L.llmdot_cuda_kvq_attention(p, b, attn(), P, 256, P, 256, None, None, 0, None)]
    for call in calls:
        assert call(None, batch()) == INVALID and call(pool(), None) == INVALID
        for kw, status in BAD_POOLS:
            assert call(pool(**kw), batch()) == status, kw
            assert message().startswith("kvq_")
        for kw in BAD_BATCHES:
            assert call(pool(), batch(**kw)) == INVALID, kw


def test_row_refusals():
    L = native.lib()
    for call in (L.llmdot_cuda_kvq_write, L.llmdot_cuda_kvq_read):
        p, b = pool(), batch(rows=3)
        assert call(p, b, P, P, 12, 128, 128, None) == UNSUPPORTED          # a quantised ggml type
        assert call(p, b, None, P, 1, 128, 128, None) == INVALID
        assert call(p, b, P, P, 1, 127, 128, None) == INVALID               # rows overlap
        assert call(p, b, P + 1, P, 1, 128, 128, None) == INVALID           # not aligned to fp16
        assert call(p, batch(rows=0), None, None, 1, 0, 0, None) == 0       # nothing to do


def test_attention_refusals():
    L = native.lib()
    need = C.c_size_t()
    for kw, status in [(dict(type=8), UNSUPPORTED), (dict(heads=3), INVALID), (dict(heads=0), INVALID), (dict(prefix_len=-1), INVALID),
                       (dict(prefix_len=64), INVALID), (dict(window=-1), INVALID), (dict(scale=float("nan")), INVALID),
                       (dict(softcap=-1.0), INVALID), (dict(softcap=float("inf")), INVALID)]:
        assert L.llmdot_cuda_kvq_attention_workspace(pool(), batch(), attn(**kw), need) == status, kw
        assert L.llmdot_cuda_kvq_attention(pool(), batch(), attn(**kw), P, 256, P, 256, None, P, 1 << 30, None) == status, kw
    b = batch(rows=2)
    assert L.llmdot_cuda_kvq_attention(pool(), b, attn(), None, 256, P, 256, None, P, 1 << 30, None) == INVALID
    assert L.llmdot_cuda_kvq_attention(pool(), b, attn(), P, 255, P, 256, None, P, 1 << 30, None) == INVALID
    assert L.llmdot_cuda_kvq_attention(pool(), b, attn(), P + 1, 256, P, 256, None, P, 1 << 30, None) == INVALID
    assert L.llmdot_cuda_kvq_attention_workspace(pool(), b, attn(), None) == INVALID
    assert L.llmdot_cuda_kvq_attention(pool(), batch(rows=0), attn(), None, 0, None, 0, None, None, 0, None) == 0


def test_verify_refusals():
    L = native.lib()

    def args(**kw):
        d = dict(batch=1, drafts=2, vocab=100, p=P, q=P, ld_p=100, ld_q=100, draft=P, uniform=P, n_draft=None, tokens=P, accepted=P)
        d.update(kw)
        return native.Verify(**d)

    assert L.llmdot_cuda_verify_draft(None, None) == INVALID
    for kw, status in [(dict(batch=-1), INVALID), (dict(drafts=-1), INVALID), (dict(vocab=0), INVALID), (dict(drafts=65), UNSUPPORTED),
                       (dict(vocab=(1 << 22) + 1, ld_p=1 << 23, ld_q=1 << 23), UNSUPPORTED), (dict(p=None), INVALID),
                       (dict(draft=None), INVALID), (dict(uniform=None), INVALID), (dict(tokens=None), INVALID),
                       (dict(accepted=None), INVALID), (dict(ld_p=99), INVALID), (dict(ld_q=99), INVALID), (dict(p=P + 2), INVALID)]:
        assert L.llmdot_cuda_verify_draft(args(**kw), None) == status, kw
        assert message().startswith("verify_draft")
    assert L.llmdot_cuda_verify_draft(args(batch=0), None) == 0


def test_structs_have_the_headers_layout(tmp_path):
    names = [("llmdot_kvq_pool", native.KvqPool), ("llmdot_kvq_batch", native.KvqBatch), ("llmdot_kvq_attn", native.KvqAttn),
             ("llmdot_verify", native.Verify)]
    body = "".join(f'printf("%zu ", sizeof({n})); ' for n, _ in names)
    body += "".join(f'printf("%zu ", offsetof({n}, {f[0]})); ' for n, s in names for f in s._fields_)
    src = tmp_path / "layout.c"
    src.write_text(f'#include "{native.HEADER}"\n#include <stdio.h>\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", "-std=c99", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True).stdout.split()))
    want = [C.sizeof(s) for _, s in names] + [getattr(s, f[0]).offset for _, s in names for f in s._fields_]
    assert got == want


def test_serving_refuses_host_tensors():
    import torch

    from dotllm_b200 import serving
    k = torch.zeros(2, 2, 64, 64, dtype=torch.int8)
    s = torch.zeros(2, 2, 64)
    with pytest.raises(ValueError):
        serving.KvqPool(k, k, s, s)
    with pytest.raises(ValueError):
        serving.KvqBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), 1)
    with pytest.raises(ValueError):
        serving.verify_draft(torch.zeros(1, 1, 8), None, torch.zeros(1, 0, dtype=torch.int32), torch.zeros(1, 1))


class OnDevice:
    """A host tensor that says it is on device 0: what a call would hand to the library, without a device."""
    is_cuda = True

    def __init__(self, t):
        self.t, self.shape, self.dtype = t, t.shape, t.dtype

    def dim(self):
        return self.t.dim()

    def stride(self):
        return self.t.stride()

    def is_contiguous(self):
        return self.t.is_contiguous()

    def get_device(self):
        return 0

    def data_ptr(self):
        return self.t.data_ptr()

    def new_empty(self, *a, **kw):
        return OnDevice(self.t.new_empty(*a, **kw))


@pytest.fixture
def launches(monkeypatch):
    """The arguments of the library calls that would have been made."""
    from dotllm_b200 import serving
    made = []
    monkeypatch.setattr(serving, "lib", lambda: type("L", (), {"llmdot_cuda_verify_draft": None})())
    monkeypatch.setattr(serving, "_call", lambda fn, device, *args: made.append(args))
    return made


def rows_end(start, rows, ld, vocab):
    """Address behind the last row that the kernel may read."""
    return start + 4 * ((rows - 1) * ld + vocab)


def test_verify_reads_stay_inside_their_tensors(launches):
    """Whatever strides are accepted, row b * n + i of the call is row (b, i) of the tensor, and the last ends inside it."""
    import torch

    from dotllm_b200 import serving
    B, V = 5, 12
    flat = torch.rand(B * 4 * (V + 3))

    def views(n):
        yield flat[:B * n * V].view(B, n, V)                                     # dense
        yield flat.view(B, 4, V + 3)[:, :n, :V] if n in (1, 4) else flat[:B * n * (V + 3)].view(B, n, V + 3)[..., :V]  # wide rows
        yield flat.view(B, 4, V + 3)[:, :n, 1:V + 1]                             # some of each sequence's rows
        yield flat[:V].expand(B, n, V)                                           # one row for all
        yield flat[-V:].expand(B, n + 1, V)[:, :n]                               # the same, every stride between rows 0
        yield flat[:B * V].view(B, 1, V).expand(B, n, V)                         # one row per sequence
        yield flat[:n * V].view(1, n, V).expand(B, n, V)                         # the same rows for all sequences
        yield flat[:B * n * V].view(n, B, V).transpose(0, 1)

    for k in (0, 1, 3):
        draft, u = OnDevice(torch.zeros(B, k, dtype=torch.int32)), OnDevice(torch.rand(B, k + 1))
        for p in views(k + 1):
            for q in [None] if k == 0 else [None, *views(k)]:
                launches.clear()
                try:
                    serving.verify_draft(OnDevice(p), None if q is None else OnDevice(q), draft, u)
                except ValueError:
                    continue
                a = launches[0][0]
                for t, start, ld, n in [(p, a.p, a.ld_p, k + 1)] + ([] if q is None else [(q, a.q, a.ld_q, k)]):
                    assert rows_end(start, B * n, ld, V) <= t.untyped_storage().data_ptr() + t.untyped_storage().nbytes(), (t.shape, t.stride())
                    for b in range(B):
                        for i in range(n):
                            assert start + 4 * (b * n + i) * ld == t[b, i].data_ptr(), (t.shape, t.stride())


def test_verify_takes_evenly_strided_rows_and_refuses_shared_ones(launches):
    import torch

    from dotllm_b200 import serving
    B, V = 5, 12

    def call(p, q):
        k = p.shape[1] - 1
        serving.verify_draft(OnDevice(p), None if q is None else OnDevice(q), OnDevice(torch.zeros(B, k, dtype=torch.int32)),
                             OnDevice(torch.rand(B, k + 1)))

    call(torch.rand(B, 4, V)[:, :1], None)   # one row of several
    call(torch.rand(B, 4, V)[:, -1:], None)
    call(torch.rand(B, 2, V), torch.rand(B, 3, V)[:, 1:2])
    call(torch.rand(B, 2, V + 4)[..., :V], torch.rand(B, V).unsqueeze(1))
    for p, q in [(torch.rand(V).expand(B, 1, V), None), (torch.rand(V).expand(B, 2, V)[:, :1], None),
                 (torch.rand(B, 2, V), torch.rand(V).expand(B, 2, V)[:, 1:]), (torch.rand(B, 2, V), torch.rand(V).expand(B, 1, V)),
                 (torch.rand(B, 2, V), torch.rand(1, 1, V).expand(B, 1, V)), (torch.rand(1, 2, V).expand(B, 2, V), None),
                 (torch.rand(B, 4, V)[:, :2], None)]:
        with pytest.raises(ValueError):
            call(p, q)


def workspace(batch_kw, attn_kw, pool_kw=()):
    need = C.c_size_t()
    status = native.lib().llmdot_cuda_kvq_attention_workspace(pool(**dict(pool_kw)), batch(**batch_kw), attn(**attn_kw), need)
    return status, need.value


def test_a_loose_max_rows_changes_nothing():
    """max_rows is a bound: no sequence has more rows than the call, so one above that is the same bound."""
    for heads, hk, typ in ((32, 8, 25), (8, 1, 0), (65536, 1, 0), (4, 4, 1)):
        for rows, prefix in ((4, 0), (3, 500), (64, 70)):
            kw = dict(rows=rows, max_pages=300)
            a = dict(heads=heads, type=typ, prefix_len=prefix, prefix_pages=P)
            tight = workspace(dict(kw, max_rows=rows), a, dict(heads_kv=hk))
            assert tight[0] == 0
            for loose in (rows + 1, 1000, 1 << 20, 2 ** 31 - 1):
                assert workspace(dict(kw, max_rows=loose), a, dict(heads_kv=hk)) == tight, (heads, rows, loose)


def test_too_many_blocks_are_refused():
    """The largest counts that the checks let through, together: more blocks than a launch has, refused before one."""
    L = native.lib()
    p, a = pool(heads_kv=4096, n_pages=1), attn(heads=4096, type=0)
    for n, m in ((2 ** 31 - 1, 1 << 24), (1 << 30, 1 << 18), (1 << 20, 1 << 24)):
        b = batch(batch=n, rows=2, max_rows=2 ** 31 - 1, max_pages=m)
        assert L.llmdot_cuda_kvq_attention(p, b, a, P, 4096 * 64, P, 4096 * 64, None, P, 1 << 60, None) == INVALID, (n, m)
        assert "too many" in message()


@pytest.mark.parametrize("typ", [0, 1, 25])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("prefix", [0, 5000, 500000])
def test_scratch_is_bounded(typ, dim, prefix):
    """Prefix and own pages leave at most 128 MB of partial results each, or those of one chunk where a call has so many
    rows that one takes more, whatever the table's length and the types."""
    for heads, hk in ((32, 8), (32, 32), (8, 1)):
        for n, rows in ((1, 1), (1, 200), (1, 2048), (1, 8192), (96, 480), (64, 64)):
            for pages in (1, 32, 256, 2048, 1 << 16):
                chunk = rows * heads * (4 * dim + 8)
                status, size = workspace(dict(batch=n, rows=rows, max_rows=-(-rows // n), max_pages=pages),
                                         dict(heads=heads, type=typ, prefix_len=prefix, prefix_pages=P), dict(heads_kv=hk, head_dim=dim))
                assert status == 0 and size <= 2 * max(chunk, 128 << 20), (heads, hk, rows, pages, size)


def test_counts_beyond_32_bits_are_not_cut(monkeypatch):
    """The library's counts are 32-bit: a larger one reaches it as the largest, never as what its low bits happen to be."""
    import torch

    from dotllm_b200 import serving
    made = []
    monkeypatch.setattr(serving, "_call", lambda fn, device, *args: made.append(args))
    codes = OnDevice(torch.zeros(2, 2, 64, 64, dtype=torch.int8))
    scales = OnDevice(torch.zeros(2, 2, 64))
    p = serving.KvqPool(codes, codes, scales, scales)

    def ints(*shape):
        return OnDevice(torch.zeros(*shape, dtype=torch.int32))

    q = OnDevice(torch.zeros(3, 4, 64))
    for big in (2 ** 31, 2 ** 32, 2 ** 32 + 10, 2 ** 40 + 1):
        b = serving.KvqBatch(ints(2), ints(1), ints(1, 2), big)
        serving.kvq_attention(p, b, q, window=big)
        assert made[-1][1].max_rows == 2 ** 31 - 1 and made[-1][2].window == 2 ** 31 - 1
        b = serving.KvqBatch(ints(2), ints(1), ints(1, 2), 3)
        for kw in (dict(window=-big), dict(prefix_len=-big)):
            with pytest.raises(native.CudaBackendError):
                serving.kvq_attention(p, b, q, **kw)
    wide = OnDevice(torch.zeros(1).expand(1, 1, 2 ** 32 + 5))  # (refused by its stride otherwise)
    monkeypatch.setattr(OnDevice, "stride", lambda self: (2 ** 32 + 5, 2 ** 32 + 5, 1) if self is wide else self.t.stride())
    serving.verify_draft(wide, None, ints(1, 0), OnDevice(torch.zeros(1, 1)))
    assert made[-1][0].vocab == 2 ** 31 - 1


def test_misaligned_pointers_are_refused():
    """Lengths, lists, numbers and results off their type's boundary never reach the device."""
    L = native.lib()
    need = C.c_size_t()
    for kw in (dict(row_start=P + 1), dict(seq_len=P + 2), dict(pages=P + 3)):
        b = batch(**kw)
        assert L.llmdot_cuda_kvq_write(pool(), b, P, P, 1, 128, 128, None) == INVALID, kw
        assert L.llmdot_cuda_kvq_read(pool(), b, P, P, 1, 128, 128, None) == INVALID, kw
        assert L.llmdot_cuda_kvq_attention_workspace(pool(), b, attn(), need) == INVALID, kw
    a = attn(prefix_len=64, prefix_pages=P + 2)
    assert L.llmdot_cuda_kvq_attention_workspace(pool(), batch(), a, need) == INVALID
    assert L.llmdot_cuda_kvq_attention(pool(), batch(), attn(), P, 256, P, 256, P + 2, P, 1 << 30, None) == INVALID
    assert "aligned" in message()
    ok = dict(batch=1, drafts=2, vocab=100, p=P, q=P, ld_p=100, ld_q=100, draft=P, uniform=P, n_draft=None, tokens=P, accepted=P)
    for name in ("p", "q", "draft", "uniform", "n_draft", "tokens", "accepted"):
        assert L.llmdot_cuda_verify_draft(native.Verify(**dict(ok, **{name: P + 2})), None) == INVALID, name
        assert "aligned" in message()
