"""GPU: weights and scales that the groups share, through the binding."""
import pytest

from test_gpu_products import generator, offsets_of, scaled, whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [[0, 1, 0, 2, 1], [0, 50, 0, 2, 50], [700, 0, 1300, 60, 9], [3]])
@pytest.mark.parametrize("scales", ["expanded", "apart", "overlapping", "a group's own"])
def test_8_bit_groups_that_share_weights_and_scales(node, sizes, scales):
    import torch
    gen, groups, m, k = generator(73), len(sizes), 130, 264
    n = sum(sizes)
    A, B = whole(gen, 1, m, k).expand(groups, m, k), whole(gen, n, k)
    if scales == "expanded":
        sa = torch.rand(m, generator=gen, device="cuda").expand(groups, m)
    elif scales == "apart":
        sa = torch.rand(groups, m + 7, generator=gen, device="cuda")[:, :m]
    elif scales == "overlapping":
        sa = torch.rand(m + groups, generator=gen, device="cuda").unfold(0, m, 1)[:groups]
    else:
        sa = torch.rand(groups, m, generator=gen, device="cuda")
    sb = torch.rand(n, generator=gen, device="cuda")
    C = torch.empty(n, m, device="cuda")
    assert node.grouped_gemm_i8_device(offsets_of(sizes), A, sa, B, sb, C) == 0
    at = 0
    for g, s in enumerate(sizes):
        sums = B[at:at + s].double() @ A[g].double().T.contiguous()
        assert torch.equal(C[at:at + s], scaled(sums, sa[g], sb[at:at + s], torch.float32)), g
        at += s


def test_scales_that_are_not_vectors_are_refused(node):
    import torch
    off = offsets_of([2, 2])
    A, B = torch.zeros(2, 6, 8, dtype=torch.int8, device="cuda"), torch.zeros(4, 8, dtype=torch.int8, device="cuda")
    C, sb = torch.zeros(4, 6, device="cuda"), torch.zeros(4, device="cuda")
    for sa in (torch.zeros(6, 2, device="cuda").T, torch.zeros(2, 12, device="cuda")[:, ::2], torch.zeros(2, 1, device="cuda").expand(2, 6), torch.zeros(1, 6, device="cuda"),
               torch.zeros(6, device="cuda")):
        with pytest.raises(ValueError):
            node.grouped_gemm_i8_device(off, A, sa, B, sb, C)
