"""GPU: every variant of the products' tiles, whatever the rules that choose among them: tile, feed and slices are forced through the
test-support library, with several tiles a workgroup, inner lengths that cut a chunk in the first, a middle and the last k-tile, and
sums that are added to what is there; and the rounding to 8 bits at the lengths where its kernels change.  Bounds as in test_gpu_products.py."""
import numpy as np
import pytest

from helpers import U
from test_gpu_products import check_outer, check_product, generator, kind, offsets_of, scaled, whole

pytestmark = pytest.mark.gpu

# more tiles of every size than workgroups fit the chip: 1000 tiles of 128 x 128, 300 of 256 x 256 with 2056 rows
MANY = [1000, 0, 3000, 2100, 77, 2500]
DIRECT, STAGED = ((0, 0, 0), (0, 0, 0)), ((1, 3, 5), (1, 0, 3))


@pytest.fixture(scope="module")
def library(node):
    lib = node.lib.load_test_hooks()
    for name, (res, args) in node.lib.SIGNATURES.items():
        f = getattr(lib, name)
        f.restype, f.argtypes = res, args
    lib.starneig_node_init(1, 1, node.NO_MESSAGES)
    yield lib
    lib.starneig_node_finalize()


@pytest.fixture
def forced(node, library, monkeypatch):
    """force(tile, slices): the binding's products run in the test-support library with this choice."""
    monkeypatch.setattr(node.lib, "_lib", library)

    def force(tile, slices=1):
        library.sn_internal_product_force(tile, slices)
    yield force
    library.sn_internal_product_force(0, 0)


@pytest.mark.parametrize("type_", ["bf16", "f16"])
@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("tile,feed", [(64, DIRECT), (128, DIRECT), (256, DIRECT), (64, STAGED), (128, STAGED)])
@pytest.mark.parametrize("k", [42, 168, 301])
def test_product(node, forced, trans, type_, tile, feed, k):
    forced(tile)
    aligned = feed == DIRECT
    # (aligned columns: even leading dimensions)
    pads, shifts = ((k % 2 if trans == "T" else 0, k % 2, 0), feed[1]) if aligned else feed
    check_product(node, trans, type_, MANY, 2056 + 2 * aligned, k, first=2, behind=3, pads=pads, shifts=shifts)
    check_product(node, trans, type_, [3, 0, 17, 1], 34, k, first=2, behind=3, pads=pads, shifts=shifts)


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 2, 3, 4])
def test_product_of_hardly_any_rows(node, forced, trans, tile, m):
    """Leading dimensions smaller than a chunk, inner lengths just past a k-tile."""
    forced(tile)
    for k in (63, 64, 65, 66, 67, 129, 130):
        check_product(node, trans, "bf16", [5, 0, 70], m, k, pads=(k % 2 if trans == "T" else m % 2, k % 2, 0))


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tile,pad,shift", [(64, 0, 0), (128, 0, 0), (256, 0, 0), (64, 3, 5), (128, 3, 5)])
@pytest.mark.parametrize("k", [42, 333, 400])
def test_8_bit_product(node, forced, out, tile, pad, shift, k):
    import torch
    forced(tile)
    pad = pad if shift else -k % 4
    for sizes, m in ((MANY, 2058), ([3, 0, 17, 1], 34)):
        gen, groups, first, behind = generator(k), len(sizes), 2, 3
        n = first + sum(sizes) + behind
        A, B = whole(gen, groups, m, k, pad=pad, shift=shift), whole(gen, n, k, pad=pad, shift=shift)
        sa, sb = torch.rand(groups, m, generator=gen, device="cuda") * 1e-2, torch.rand(n, generator=gen, device="cuda") * 1e-2
        C = torch.full((n, m + 3), 7.0, dtype=kind(out), device="cuda")
        assert node.grouped_gemm_i8_device(offsets_of(sizes, first), A, sa, B, sb, C[:, :m]) == 0
        at = first
        for g, s in enumerate(sizes):
            sums = B[at:at + s].double() @ A[g].double().T.contiguous()
            assert torch.equal(C[at:at + s, :m], scaled(sums, sa[g], sb[at:at + s], kind(out))), g
            at += s
        assert bool((C[:, m:] == 7.0).all()) and bool((C[:first] == 7.0).all()) and bool((C[n - behind:] == 7.0).all())


@pytest.mark.parametrize("type_,out", [("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("beta", [0.0, 0.5])
@pytest.mark.parametrize("slices", [1, 2, 7, 64])
@pytest.mark.parametrize("tile,feed", [(64, DIRECT), (128, DIRECT), (256, DIRECT), (64, STAGED), (128, STAGED)])
def test_outer(node, forced, type_, out, beta, slices, tile, feed):
    forced(tile, slices)
    pads, shifts = ((0, 0, 3), feed[1]) if feed == DIRECT else feed
    check_outer(node, type_, out, [300, 0, 1000, 65, 5, 777, 128, 1], 1096, 1544, beta, first=2, behind=3, pads=pads, shifts=shifts)
    # more groups than a wave has lanes; rows and columns of less than a chunk (aligned), of just one (not)
    check_outer(node, type_, out, [1] * 40 + [65, 0, 66, 130] * 8, 10, 8 + 2 * (feed == DIRECT), beta, first=1, behind=1, pads=pads, shifts=shifts)
    if feed == DIRECT:
        for m, n in ((2, 2), (2, 130), (4, 2)):
            check_outer(node, type_, out, [65, 0, 66, 129, 300], m, n, beta, pads=pads, shifts=shifts)


def test_outer_without_scratch_memory_has_the_tile_that_is_best_without(node, forced, library):
    """With scratch memory the rules take tiles of 256 here, without it those of 64, whose four parts of the sum show in the last bits."""
    import torch
    k, m, n = 36501, 1050, 666
    assert library.sn_internal_product_outer_cut(1, 1, m, n, k, 64) % 1000 != 64 and library.sn_internal_product_outer_cut(1, 1, m, n, k, 1) == 1064
    gen = generator(7)
    X, Y = (torch.randn(k, s, generator=gen, device="cuda").bfloat16() for s in (m, n))
    off, stream = offsets_of([k]), torch.cuda.current_stream().cuda_stream

    def result():
        D = torch.empty(n, m, device="cuda")
        assert library.starneig_amd_grouped_outer_device(node.AMD_BF16, node.AMD_F32, 1, m, n, k, off.data_ptr(), X.data_ptr(), m, Y.data_ptr(), n, 0.0,
                                                         D.data_ptr(), m, m * n, None, 0, stream) == 0
        return D

    by_rule, by_tile = result(), {}
    for tile in (64, 128):
        forced(tile)
        by_tile[tile] = result()
    assert torch.equal(by_rule, by_tile[64]) and not torch.equal(by_rule, by_tile[128])


@pytest.mark.parametrize("beta", [0.0, 0.5])
@pytest.mark.parametrize("slices", [1, 3, 16])
def test_f64_outer(node, forced, beta, slices):
    forced(64, slices)
    check_outer(node, "f64", "f64", [300, 0, 1000, 65, 5, 777, 128, 1], 330, 140, beta, first=2, behind=3, pads=(1, 0, 3))
    check_outer(node, "f64", "f64", [1] * 40 + [17, 0, 16, 33] * 8, 10, 7, beta, first=1, behind=1)


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("k", [1, 15, 333])
def test_f64_product(node, forced, trans, k):
    """The tile of 64 also where few outputs would take the other kernel."""
    forced(64)
    check_product(node, trans, "f64", [3, 0, 17, 1], 34, k, first=2, behind=3, pads=(1, 0, 3))


@pytest.mark.parametrize("slices", [1, 5])
def test_f64_outer_of_columns_far_apart(node, forced, slices):
    """Columns more than 4 MB apart are read by another kernel, here over several slices with empty ones among them."""
    import torch
    forced(64, slices)
    gen, sizes, m, n, ld = generator(91), [300, 0, 500, 20], 130, 70, (1 << 19) + 3
    k = sum(sizes)
    X = torch.empty(k, ld, dtype=torch.float64, device="cuda")[:, :m]
    X.copy_(torch.randn(k, m, generator=gen, device="cuda", dtype=torch.float64))
    Y = torch.randn(k, n, generator=gen, device="cuda", dtype=torch.float64)
    for beta in (0.0, 0.5):
        D = torch.ones(len(sizes), n, m, dtype=torch.float64, device="cuda")
        assert node.grouped_outer_device(offsets_of(sizes), X, Y, D, beta=beta) == 0
        for g, (x, y) in enumerate(zip(X.split(sizes), Y.split(sizes))):
            ref, mag = y.T.contiguous() @ x + beta, y.T.abs().contiguous() @ x.abs() + beta
            assert bool(((D[g] - ref).abs() <= (4 * sizes[g] + 8) * U * mag).all()), g


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("k", [1024, 1025, 2048, 2049, 4096, 4097, 5001, 8192, 8193, 32768, 32769])
def test_quantize_i8_on_both_sides_of_each_kernel(node, type_, k):
    import torch
    n = 9
    X = torch.randn(n, k, generator=generator(k), device="cuda", dtype=torch.float64).mul_(3).to(kind(type_))
    Q, scale = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    assert node.quantize_i8_device(X, Q, scale) == 0
    x = X.float().cpu().numpy()
    s = np.abs(x).max(axis=1) / np.float32(127)
    assert np.array_equal(scale.cpu().numpy(), s)
    assert np.array_equal(Q.cpu().numpy(), np.rint(x / s[:, None]).astype(np.int8))


@pytest.mark.parametrize("type_", ["bf16", "f32"])
@pytest.mark.parametrize("k", [300, 5001, 33000])
def test_quantize_i8_of_tiny_and_huge_columns(node, type_, k):
    """Maxima from the smallest subnormal, where the quotient passes 127 and is limited, over the ends of the range in which the quotient comes from the
    reciprocal (scales of 2^-100 and 2^100), to the largest number."""
    import torch
    dtype = kind(type_)
    step = float(torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)           # the smallest subnormal
    tops = [step * j for j in (1, 63, 64, 127, 190, 191, 254, 255, 317, 318, 1000, 12345)]
    tops += [127 * 2.0 ** e * f for e in (-127, -126, -125, -101, -100, -99, 99, 100, 101, 120) for f in (1 - 2 ** -7, 1.0, 1 + 2 ** -7)]
    tops += [torch.finfo(dtype).max]
    gen = generator(k)
    X = torch.rand(len(tops), k, generator=gen, device="cuda", dtype=torch.float64).mul_(2).sub_(1)
    X[:, k // 2] = 1.0
    X = (X * torch.tensor(tops, dtype=torch.float64, device="cuda")[:, None]).to(dtype)
    Q, scale = torch.full((len(tops), k), 99, dtype=torch.int8, device="cuda"), torch.empty(len(tops), device="cuda")
    assert node.quantize_i8_device(X, Q, scale) == 0
    x = X.float().cpu().numpy()
    s = np.abs(x).max(axis=1) / np.float32(127)
    assert np.array_equal(scale.cpu().numpy(), s)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s[:, None] > 0, np.clip(np.rint(x / s[:, None]), -127, 127), 0)
    assert np.array_equal(Q.cpu().numpy(), q.astype(np.int8))
    # some of them are limited, in fp32 only: the smallest bf16 has a scale of 516 smallest fp32 subnormals, which half of one moves by less than a thousandth
    assert (np.abs(x).max(axis=1)[s > 0] / s[s > 0] > 127.5).any() == (type_ == "f32")


LATER = {
    "none": lambda sizes: [0] * (len(sizes) + 1),                       # every group empty
    "behind": lambda sizes: [sum(sizes)] * (len(sizes) + 1),
    "one": lambda sizes: [0] * len(sizes) + [sum(sizes) - 1],           # one group, a column less
    "reversed": lambda sizes: [0, *(sum(sizes[:-g - 2:-1]) for g in range(len(sizes)))],
}


@pytest.mark.parametrize("later", list(LATER))
@pytest.mark.parametrize("type_,tile,k,shift", [
    ("bf16", 0, 200, 0), ("bf16", 0, 5, 1), ("bf16", 64, 200, 0), ("f16", 128, 200, 0), ("bf16", 256, 200, 0), ("bf16", 64, 200, 1), ("bf16", 128, 200, 1),
    ("i8", 0, 200, 0), ("i8", 0, 5, 1), ("i8", 64, 200, 0), ("i8", 128, 200, 0), ("i8", 256, 200, 0), ("i8", 64, 201, 1), ("i8", 128, 201, 1),
    ("f64", 0, 200, 0), ("f64", 64, 200, 0), ("f64", 64, 200, -1)])
def test_offsets_that_change_during_a_call(node, forced, library, type_, tile, k, shift, later):
    """More than 64 groups, whose offsets are walked over again for every tile, and are others then: nothing is promised about the columns of C, but
    nothing else is written, and where no group has a column any more, nothing at all.  (shift -1: columns more than 4 MB apart.)"""
    import torch
    forced(tile)
    sizes = [1] * 50 + [0, 3, 0, 0, 9] * 12 + [40]
    groups, n, m, pad = len(sizes), sum(sizes), 150, 4
    counted = offsets_of(sizes)
    both = torch.cat([counted, torch.tensor(LATER[later](sizes), dtype=torch.int32, device="cuda")])
    dtype = {"i8": torch.int8}.get(type_) or kind(type_)
    one = lambda rows: torch.ones(rows * k + 1, dtype=dtype, device="cuda")[max(shift, 0):][:rows * k].view(rows, k)
    A, B = one(m)[None].expand(groups, m, k), one(n)
    if shift < 0:
        far = torch.empty(n, (1 << 19) + 3, dtype=dtype, device="cuda")
        B = far[:, :k].fill_(1)
    C = torch.full((n + 2 * pad, m + pad), 7.0, dtype=torch.float32 if type_ == "i8" else dtype, device="cuda")
    inner = C[pad:-pad, :m]
    scale = torch.ones(max(n, m), device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    assert library.sn_internal_product_later_offsets(groups + 1) == 0
    try:
        if type_ == "i8":
            assert library.starneig_amd_grouped_gemm_i8_device(
                node.AMD_F32, groups, m, n, k, both.data_ptr(), A.data_ptr(), k, 0, scale.data_ptr(), 0, B.data_ptr(), k, scale.data_ptr(),
                inner.data_ptr(), m + pad, stream) == 0
        else:
            assert node.grouped_gemm_device("T", both[:groups + 1], A, B, inner) == 0
        torch.cuda.synchronize()
    finally:
        assert library.sn_internal_product_later_offsets(0) == 0
    if later in ("none", "behind"):
        assert bool((inner == 7.0).all())
    else:
        assert bool(((inner == 7.0) | (inner == float(k))).all())
    inner.fill_(7.0)
    assert bool((C == 7.0).all())
