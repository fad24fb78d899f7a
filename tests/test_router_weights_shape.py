"""Router weights come as [tokens, top-k], or flat in that order; as many numbers in another shape would be other pairs' weights."""
import pytest
import torch


def test_slots_first_is_refused():
    from gridbook_b200 import kernels
    place = torch.zeros(6, dtype=torch.int32)
    srt = kernels.MoESort(place, place, place, place, 2)
    y = torch.zeros(6, 16)
    for w in (torch.ones(2, 3), torch.ones(1, 6), torch.ones(3, 3), torch.ones(5), torch.ones(6, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="router weight"):
            kernels.moe_unpermute(y, srt, w)
    for w in (torch.ones(3, 2), torch.ones(6), torch.ones(6, 1)):          # these get as far as the device check
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            kernels.moe_unpermute(y, srt, w)


@pytest.mark.gpu
def test_shapes_that_say_the_same():
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(3)
    E, H, inter, T, topk = 4, 128, 128, 6, 2
    w13 = torch.randn(E, 2 * inter, H, generator=g, device=dev).to(torch.float8_e4m3fn)
    w2 = torch.randn(E, H, inter, generator=g, device=dev).to(torch.float8_e4m3fn)
    s13, s2 = torch.full((E, 2, 1), 0.1, device=dev), torch.full((E, 1, 1), 0.1, device=dev)
    x = torch.randn(T, H, generator=g, device=dev)
    ids = torch.rand(T, E, generator=g, device=dev).topk(topk, -1)[1]
    w = torch.rand(T, topk, generator=g, device=dev)
    want = kernels.moe_fp8_blocks(x, w13, s13, w2, s2, w, ids)
    for same in (w.reshape(-1), w.reshape(-1, 1), w.view(2, 3, topk)):
        assert torch.equal(kernels.moe_fp8_blocks(x, w13, s13, w2, s2, same, ids), want)
    with pytest.raises(RuntimeError, match="router weights"):
        kernels.moe_fp8_blocks(x, w13, s13, w2, s2, w.t().contiguous(), ids)
    srt = kernels.moe_sort(ids, E)
    rows = kernels.moe_permute(x, srt)
    assert torch.equal(kernels.moe_unpermute(rows, srt, w.reshape(-1)), kernels.moe_unpermute(rows, srt, w))
    with pytest.raises(RuntimeError, match="router weights"):
        kernels.moe_unpermute(rows, srt, w.t())
