"""Which rows of their tensors the serving operators take: slices of wider tensors give what dense copies give."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 33, 1000])
def test_verify_takes_one_row_of_several(gpu, V):
    """One draft, or none, per sequence: the rows are a sequence apart, whatever lies between them."""
    import torch
    from dotllm_b200 import serving
    g = torch.Generator("cuda").manual_seed(V)
    p, q = (torch.softmax(2 * torch.randn(7, 3, V, device="cuda", generator=g), -1) for _ in range(2))
    draft = torch.randint(0, V, (7, 1), device="cuda", generator=g, dtype=torch.int32)
    u = torch.rand(7, 2, device="cuda", generator=g)
    for i in range(3):
        for a, b in ((serving.verify_draft(p[:, :2].contiguous(), q[:, i:i + 1], draft, u),
                      serving.verify_draft(p[:, :2].contiguous(), q[:, i:i + 1].contiguous(), draft, u)),
                     (serving.verify_draft(p[:, i:i + 1], None, draft[:, :0].contiguous(), u[:, 1:].contiguous()),
                      serving.verify_draft(p[:, i:i + 1].contiguous(), None, draft[:, :0].contiguous(), u[:, 1:].contiguous()))):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_verify_refuses_one_row_for_all_sequences(gpu):
    import torch
    from dotllm_b200 import serving
    p, one = torch.rand(4, 2, 50, device="cuda"), torch.rand(50, device="cuda")
    draft, u = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.rand(4, 2, device="cuda")
    for q in (one.expand(4, 1, 50), one.expand(4, 2, 50)[:, 1:], one.view(1, 1, 50).expand(4, 1, 50)):
        with pytest.raises(ValueError):
            serving.verify_draft(p, q, draft, u)
        serving.verify_draft(p, q.contiguous(), draft, u)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads", [4, 48])
def test_a_loose_max_rows_gives_the_same_bits(gpu, typ, heads):
    import torch
    from dotllm_b200 import serving
    g = torch.Generator("cuda").manual_seed(5)
    pool = serving.KvqPool.empty(8, 2, 64)
    pages = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = torch.tensor([200, 130], dtype=torch.int32, device="cuda")
    all_rows = torch.tensor([0, 200, 330], dtype=torch.int32, device="cuda")
    serving.kvq_write(pool, serving.KvqBatch(all_rows, lens, pages, 200),
                      *(torch.randn(330, 2, 64, device="cuda", generator=g) for _ in range(2)))
    row_start = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    q = torch.randn(5, heads, 64, device="cuda", generator=g).to(getattr(torch, typ))
    want = serving.kvq_attention(pool, serving.KvqBatch(row_start, lens, pages, 5), q)
    for loose in (6, 1000, 2 ** 31 - 1):
        assert torch.equal(serving.kvq_attention(pool, serving.KvqBatch(row_start, lens, pages, loose), q), want)
