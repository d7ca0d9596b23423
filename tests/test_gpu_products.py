"""GPU: products over ragged groups of columns and in 8-bit integers, against plain 64-bit products.

Tolerances.  The product of two bf16 or fp16 numbers is exact in fp32 (16 or 22 bits).  A sum of k of them in fp32, in any order and
with each addition off by at most a whole step (2^-23 of the partial sum, which is at most the sum of the magnitudes),
is off by at most k 2^-23 sum |a b|; the rounding to the result's type adds half a step, eps / 2 |value|, or half of the smallest
subnormal.  fp64: 4 k u sum |a b| like the library's other products.  8-bit sums are exact, and the scaling is three
fp32 roundings that torch does in the same order: equal bits."""
import numpy as np
import pytest

from helpers import U

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "f16", "f64"]


def kind(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}[name]


def generator(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def padded(gen, *shape, dtype, pad=0, shift=0, scale=1.0, fill=float("nan")):
    """A tensor whose rows lie `pad` entries apart, `shift` entries behind an aligned address; NaN in between."""
    import torch
    full = torch.full((int(np.prod(shape[:-1])) * (shape[-1] + pad) + shift,), fill, dtype=dtype, device="cuda")
    view = full[shift:].view(*shape[:-1], shape[-1] + pad)[..., : shape[-1]]
    view.copy_(torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * scale)
    return view


def offsets_of(sizes, first=0):
    import torch
    return torch.tensor(np.concatenate([[first], first + np.cumsum(sizes)]), dtype=torch.int32, device="cuda")


def half_step(value, dtype):
    import torch
    if dtype == torch.float64:
        return 0 * value.abs()
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) * (1 + 2 ** -10) + info.smallest_normal * info.eps / 2


def product_bound(k, magnitude, value, dtype):
    import torch
    unit = 4 * U if dtype == torch.float64 else 2.0 ** -23
    return k * unit * magnitude + half_step(value, dtype)


def check_product(S, trans, type_, sizes, m, k, first=0, behind=0, pads=(0, 0, 0), shifts=(0, 0, 0), share=False, seed=1):
    import torch
    gen, dtype, groups, n = generator(seed), kind(type_), len(sizes), first + sum(sizes) + behind
    shape = (m, k) if trans == "T" else (k, m)
    A = padded(gen, 1 if share else groups, *shape, dtype=dtype, pad=pads[0], shift=shifts[0], scale=k ** -0.5)
    if share:
        A = A.expand(groups, *shape)
    B = padded(gen, n, k, dtype=dtype, pad=pads[1], shift=shifts[1])
    C = padded(gen, n, m, dtype=dtype, pad=pads[2], shift=shifts[2], fill=7.0)
    # the columns of no group hold NaN and must neither be written nor leak into others
    B[:first] = float("nan"); B[n - behind:] = float("nan")
    before = C.clone()
    storage = C.untyped_storage()
    raw = torch.empty(0, dtype=dtype, device="cuda").set_(storage)
    raw_before = raw.clone()
    assert S.grouped_gemm_device(trans, offsets_of(sizes, first), A, B, C) == 0
    at = first
    for g, s in enumerate(sizes):
        a, b = A[g].double(), B[at:at + s].double()
        a = a.T if trans == "T" else a
        ref = b @ a
        bound = product_bound(k, b.abs() @ a.abs(), ref, dtype)
        off = (C[at:at + s].double() - ref).abs()
        assert bool((off <= bound).all()), (g, s, float((off - bound).max()))
        at += s
    assert torch.equal(C[:first], before[:first]) and torch.equal(C[n - behind:], before[n - behind:])
    # and nothing beside the matrix
    C.copy_(before)
    assert torch.equal(raw, raw_before)


SIZES = [
    # (sizes of the groups, m, k)
    ([1], 1, 1),
    ([0, 1, 0], 5, 3),
    ([7], 64, 64),
    ([3, 0, 17, 1], 33, 65),
    ([64, 64], 64, 128),
    ([130, 1, 0, 255, 63], 129, 257),
    ([16, 15, 17], 300, 1000),
    ([700], 257, 96),
    ([257, 513, 5], 512, 512),
    ([2000, 31], 384, 640),
    ([1] * 70 + [5, 0, 0, 9] * 20, 96, 72),         # more groups than a wave has lanes
    ([0] * 64 + [3] + [0] * 63 + [40], 40, 136),
    ([1000, 0, 5000, 2100, 77], 2056, 168),         # enough tiles to fill the chip: the large ones
    ([1000, 0, 5000, 2100, 77], 2058, 42),          # inner lengths that end within a chunk of 8, in the first and the second k-tile
    ([1000, 0, 5000, 2100, 77], 2058, 108),
    ([70, 0, 3], 6, 6),
    ([300], 2, 2),
    ([200, 30], 130, 204),
]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("sizes,m,k", SIZES)
def test_product(node, trans, type_, sizes, m, k):
    check_product(node, trans, type_, sizes, m, k)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("pads,shifts", [((8, 8, 8), (0, 0, 0)), ((1, 3, 5), (0, 0, 0)), ((0, 0, 0), (1, 3, 5)), ((2, 4, 6), (4, 2, 1))])
@pytest.mark.parametrize("sizes,m,k", [([3, 0, 170, 1], 133, 203), ([300, 20], 264, 328), ([1, 2], 520, 1336)])
def test_product_strides_and_alignment(node, trans, type_, pads, shifts, sizes, m, k):
    check_product(node, trans, type_, sizes, m, k, first=2, behind=3, pads=pads, shifts=shifts)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("trans", ["T", "N"])
def test_product_one_matrix_for_all_groups(node, trans, type_):
    check_product(node, trans, type_, [5, 0, 40, 3], 72, 80, share=True)


@pytest.mark.parametrize("type_", TYPES)
def test_product_without_inner_terms_is_zero(node, type_):
    import torch
    A = torch.empty(2, 6, 0, dtype=kind(type_), device="cuda")
    B = torch.empty(5, 0, dtype=kind(type_), device="cuda")
    C = torch.full((5, 6), 3.0, dtype=kind(type_), device="cuda")
    assert node.grouped_gemm_device("T", offsets_of([2, 1], 1), A, B, C) == 0
    assert C.tolist() == [[3.0] * 6] + [[0.0] * 6] * 3 + [[3.0] * 6]
    D = torch.full((2, 6, 4), 3.0, dtype=kind(type_), device="cuda")
    X = torch.empty(0, 4, dtype=kind(type_), device="cuda")
    Y = torch.empty(0, 6, dtype=kind(type_), device="cuda")
    assert node.grouped_outer_device(offsets_of([0, 0]), X, Y, D, beta=0.5) == 0
    assert bool((D == 1.5).all())
    assert node.grouped_outer_device(offsets_of([0, 0]), X, Y, D) == 0
    assert bool((D == 0).all())


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("offsets,spans", [
    ([-5, 4, 9], [(0, 4), (4, 9)]),                     # below zero: zero
    ([0, 4, 2000000000], [(0, 4), (4, 20)]),            # past the end: the end
    ([0, 12, 7, 15], [(0, 12), (12, 12), (12, 15)]),    # going back: an empty group
    ([9, 3, -1, 2], [(9, 9), (9, 9), (9, 9)]),
    ([-2147483648, 2147483647, -2147483648], [(0, 20), (20, 20)]),
])
def test_offsets_that_are_no_prefix_sums(node, trans, offsets, spans):
    import torch
    gen, n, m, k = generator(3), 20, 72, 40
    A = torch.randn(len(spans), m, k, generator=gen, device="cuda").bfloat16()
    if trans == "N":
        A = A.transpose(1, 2).contiguous()
    B = torch.randn(n, k, generator=gen, device="cuda").bfloat16()
    C = torch.full((n, m), 7.0, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    assert node.grouped_gemm_device(trans, off, A, B, C) == 0
    want = torch.full((n, m), 7.0, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for g, (a, b) in enumerate(spans):
        W = A[g].double().T if trans == "T" else A[g].double()
        want[a:b] = B[a:b].double() @ W
        size[a:b] = B[a:b].double().abs() @ W.abs()
    assert bool(((C.double() - want).abs() <= product_bound(k, size, want, torch.bfloat16)).all())
    D = torch.full((len(spans), m, k), 7.0, dtype=torch.float32, device="cuda")
    Y = torch.randn(n, m, generator=gen, device="cuda").bfloat16()
    assert node.grouped_outer_device(off, B, Y, D) == 0
    for g, (a, b) in enumerate(spans):
        ref = Y[a:b].double().T @ B[a:b].double()
        mag = Y[a:b].double().abs().T @ B[a:b].double().abs()
        assert bool(((D[g].double() - ref).abs() <= product_bound(n, mag, ref, torch.float32)).all())


def check_outer(S, type_, out, sizes, m, n, beta, first=0, behind=0, pads=(0, 0, 0), shifts=(0, 0, 0), seed=5):
    import torch
    gen, dtype, groups, k = generator(seed), kind(type_), len(sizes), first + sum(sizes) + behind
    X = padded(gen, k, m, dtype=dtype, pad=pads[0], shift=shifts[0])
    Y = padded(gen, k, n, dtype=dtype, pad=pads[1], shift=shifts[1], scale=0.25)
    D = padded(gen, groups, n, m, dtype=kind(out), pad=pads[2], shift=shifts[2], fill=7.0)
    X[:first] = float("nan"); X[k - behind:] = float("inf")
    Y[:first] = float("inf"); Y[k - behind:] = float("nan")
    old = D.clone()
    if beta == 0:
        D.fill_(float("nan"))           # must not be read
    raw = torch.empty(0, dtype=D.dtype, device="cuda").set_(D.untyped_storage())
    raw_before = raw.clone()
    assert S.grouped_outer_device(offsets_of(sizes, first), X, Y, D, beta=beta) == 0
    at = first
    for g, s in enumerate(sizes):
        x, y = X[at:at + s].double(), Y[at:at + s].double()
        ref, mag = y.T @ x, y.T.abs() @ x.abs()
        bound = (s * (4 * U if dtype == torch.float64 else 2.0 ** -23)) * mag
        if beta != 0:
            # beta D and its sum with the product: two more roundings of the precision that the sums are held in
            ref = ref + beta * old[g].double()
            bound = bound + (2 * U if dtype == torch.float64 else 2.0 ** -23) * (abs(beta) * old[g].double().abs() + mag)
        bound = bound + half_step(ref, D.dtype)
        off = (D[g].double() - ref).abs()
        assert bool((off <= bound).all()), (g, s, float((off - bound).max()))
        at += s
    if beta != 0:
        D.copy_(old)
    else:
        D.fill_(float("nan"))
    assert torch.equal(raw.nan_to_num(nan=-3.0), raw_before.nan_to_num(nan=-3.0))


@pytest.mark.parametrize("type_,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f64", "f64")])
@pytest.mark.parametrize("beta", [0.0, 1.0, -0.5])
@pytest.mark.parametrize("sizes,m,n", [
    ([1], 1, 1), ([0, 1, 0], 5, 3), ([33], 64, 64), ([3, 0, 17, 1], 33, 65), ([130, 1, 0, 255, 63], 129, 257), ([700], 256, 96),
    ([257, 513, 5], 300, 512), ([9000], 64, 40), ([20000], 200, 136), ([1] * 70 + [5, 0, 0, 9] * 20, 40, 72), ([4000, 60, 0, 2500], 128, 384),
    ([100, 0, 333, 64, 1] * 2, 1096, 1544),
    ([100, 0, 333, 64, 1] * 2, 1098, 1546), ([3000, 2], 6, 130), ([300], 2, 2)])
def test_outer(node, type_, out, beta, sizes, m, n):
    check_outer(node, type_, out, sizes, m, n, beta)


@pytest.mark.parametrize("type_,out", [("bf16", "f32"), ("f16", "f16"), ("f64", "f64")])
@pytest.mark.parametrize("pads,shifts", [((8, 8, 8), (0, 0, 0)), ((1, 3, 5), (0, 0, 0)), ((0, 0, 0), (1, 3, 5)), ((2, 4, 6), (4, 2, 1))])
@pytest.mark.parametrize("sizes,m,n", [([3, 0, 170, 1], 133, 203), ([300, 20], 264, 328)])
def test_outer_strides_and_alignment(node, type_, out, pads, shifts, sizes, m, n):
    check_outer(node, type_, out, sizes, m, n, 0.0, first=2, behind=3, pads=pads, shifts=shifts)
    check_outer(node, type_, out, sizes, m, n, 1.0, first=70, behind=1, pads=pads, shifts=shifts)


# ---- 8-bit integers ----------------------------------------------------------------------------------------------

def whole(gen, *shape, pad=0, shift=0, low=-127):
    import torch
    full = torch.full((int(np.prod(shape[:-1])) * (shape[-1] + pad) + shift,), -128, dtype=torch.int8, device="cuda")
    view = full[shift:].view(*shape[:-1], shape[-1] + pad)[..., : shape[-1]]
    view.copy_(torch.randint(low, 128, shape, generator=gen, device="cuda", dtype=torch.int8))
    return view


def scaled(sums, scale_row, scale_col, dtype):
    return ((sums.float() * scale_row[None, :]) * scale_col[:, None]).to(dtype)


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 3, 17), (64, 1, 64), (4096, 1, 4096), (1999, 3, 1403), (130, 16, 4096), (257, 33, 129), (300, 130, 640), (512, 512, 1024), (1000, 777, 1403),
                                   (4112, 4100, 400), (4112, 4100, 404), (300, 130, 636), (70, 90, 12)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 0), (3, 5)])
def test_gemm_i8(node, out, m, n, k, pad, shift):
    import torch
    gen = generator(m + n + k)
    A, B = whole(gen, m, k, pad=pad, shift=shift), whole(gen, n, k, pad=pad, shift=shift)
    sa, sb = torch.rand(m, generator=gen, device="cuda") * 1e-2, torch.rand(n, generator=gen, device="cuda") * 1e-2
    C = torch.full((n, m + pad), 7.0, dtype=kind(out), device="cuda")
    assert node.gemm_i8_device(A, sa, B, sb, C[:, :m]) == 0
    sums = B.double() @ A.double().T
    assert torch.equal(C[:, :m], scaled(sums, sa, sb, kind(out)))
    assert bool((C[:, m:] == 7.0).all())


def test_gemm_i8_of_the_largest_values(node):
    """k = 131071 and -128 everywhere: the sum is 2^31 - 2^14."""
    import torch
    A = torch.full((3, 131071), -128, dtype=torch.int8, device="cuda")
    B = torch.full((2, 131071), -128, dtype=torch.int8, device="cuda")
    B[1] = 127
    one = torch.ones(3, device="cuda")
    C = torch.empty(2, 3, device="cuda")
    assert node.gemm_i8_device(A, one, B, one[:2], C) == 0
    want = torch.tensor([131071 * 16384, -131071 * 16256], device="cuda").float()
    assert torch.equal(C, want[:, None].expand(2, 3))
    A0, B0 = A[:, :0], B[:, :0]
    assert node.gemm_i8_device(A0, one, B0, one[:2], C) == 0
    assert bool((C == 0).all())


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sizes,m,k", SIZES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 0), (3, 5)])
def test_grouped_gemm_i8(node, out, sizes, m, k, pad, shift):
    import torch
    gen, groups, first, behind = generator(m + k), len(sizes), 2, 3
    n = first + sum(sizes) + behind
    A, B = whole(gen, groups, m, k, pad=pad, shift=shift), whole(gen, n, k, pad=pad, shift=shift)
    sa, sb = torch.rand(groups, m, generator=gen, device="cuda") * 1e-2, torch.rand(n, generator=gen, device="cuda") * 1e-2
    C = torch.full((n, m + pad), 7.0, dtype=kind(out), device="cuda")
    assert node.grouped_gemm_i8_device(offsets_of(sizes, first), A, sa, B, sb, C[:, :m]) == 0
    at = first
    for g, s in enumerate(sizes):
        sums = B[at:at + s].double() @ A[g].double().T
        assert torch.equal(C[at:at + s, :m], scaled(sums, sa[g], sb[at:at + s], kind(out))), g
        at += s
    assert bool((C[:, m:] == 7.0).all()) and bool((C[:first] == 7.0).all()) and bool((C[n - behind:] == 7.0).all())


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 7), (2, 64), (5, 1403), (64, 4096), (1000, 520), (3, 20001), (2, 131071)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 0), (3, 5)])
def test_quantize_i8(node, type_, n, k, pad, shift):
    import torch
    gen = generator(n + k)
    X = padded(gen, n, k, dtype=kind(type_), pad=pad, shift=shift, scale=3.0)
    Q = torch.full((n, k + pad), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(n, device="cuda")
    assert node.quantize_i8_device(X, Q[:, :k], scale) == 0
    x = X.float().cpu().numpy()
    s = np.abs(x).max(axis=1) / np.float32(127)             # IEEE fp32, as numpy divides
    assert np.array_equal(scale.cpu().numpy(), s)
    assert np.array_equal(Q[:, :k].cpu().numpy(), np.rint(x / s[:, None]).astype(np.int8))
    assert bool((Q[:, k:] == 99).all())


def test_quantize_i8_of_special_columns(node):
    import torch
    X = torch.zeros(7, 300, device="cuda")
    X[1, 5] = float("nan"); X[1, 7] = 3
    X[2, 299] = float("inf"); X[2, 0] = 1
    X[3, 0] = -float("inf")
    X[4, 17] = -1e-45                       # the scale underflows
    X[5, 3] = 3.4e38; X[5, 4] = -1.7e38
    X[6] = torch.arange(300, device="cuda") - 127.0 / 2; X[6] = X[6].clamp(-127, 127)        # halves: to even
    Q = torch.full((7, 300), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(7, device="cuda")
    assert node.quantize_i8_device(X, Q, scale) == 0
    s = scale.tolist()
    assert s[0] == 0 and s[1] != s[1] and s[2] == float("inf") and s[3] == float("inf") and s[4] == 0
    assert bool((Q[:5] == 0).all())
    x = X[5, 3:5].cpu().numpy()
    assert Q[5, 3] == 127 and s[6] == 1.0
    assert Q[5, 4] == np.rint(x[1] / (x[0] / np.float32(127)))
    assert np.array_equal(Q[6].cpu().numpy(), np.rint(X[6].cpu().numpy()).astype(np.int8))
    # a column that is not finite makes its own outputs NaN, and no others
    A, sa = torch.ones(4, 300, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    C = torch.empty(7, 4, device="cuda")
    assert node.gemm_i8_device(A, sa, Q, scale, C) == 0
    assert C.isnan().all(1).tolist() == [False, True, True, True, False, False, False] and bool((C[0] == 0).all())


# ---- as they are used together -----------------------------------------------------------------------------------

def route(gen, tokens, groups, top_k):
    """Columns in the experts' order: (token of every column, offsets)."""
    import torch
    chosen = torch.randn(tokens, groups, generator=gen, device="cuda").topk(top_k, dim=1).indices.reshape(-1)
    order = chosen.sort(stable=True)
    counts = torch.bincount(chosen, minlength=groups)
    off = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    off[1:] = counts.cumsum(0)
    return order.indices // top_k, off


class Experts:
    """y = W2 relu(W1 x)^2 of every expert, its gradients by the formulas: four grouped products and two outer ones."""

    def __init__(self, S, off, W1, W2):
        self.S, self.off, self.W1, self.W2 = S, off, W1, W2

    def forward(self, x):
        import torch
        self.x = x
        self.h = torch.empty(x.shape[0], self.W1.shape[1], dtype=x.dtype, device="cuda")
        assert self.S.grouped_gemm_device("T", self.off, self.W1, x, self.h) == 0
        self.a = self.h.relu().square()
        y = torch.empty(x.shape[0], self.W2.shape[1], dtype=x.dtype, device="cuda")
        assert self.S.grouped_gemm_device("T", self.off, self.W2, self.a, y) == 0
        return y

    def backward(self, dy):
        import torch
        da, dx = torch.empty_like(self.a), torch.empty_like(self.x)
        dW1, dW2 = torch.empty_like(self.W1), torch.empty_like(self.W2)
        assert self.S.grouped_gemm_device("N", self.off, self.W2, dy, da) == 0
        assert self.S.grouped_outer_device(self.off, self.a, dy, dW2) == 0
        dh = 2 * self.h.relu() * da
        assert self.S.grouped_gemm_device("N", self.off, self.W1, dh, dx) == 0
        assert self.S.grouped_outer_device(self.off, self.x, dh, dW1) == 0
        return dx, dW1, dW2


def experts_case(dtype, seed=11, tokens=50, groups=6, d=48, hidden=72):
    import torch
    gen = generator(seed)
    token, off = route(gen, tokens, groups, 2)
    x = torch.randn(tokens, d, generator=gen, device="cuda", dtype=torch.float64).to(dtype)[token].contiguous()
    W1 = (torch.randn(groups, hidden, d, generator=gen, device="cuda", dtype=torch.float64) * d ** -0.5).to(dtype)
    W2 = (torch.randn(groups, d, hidden, generator=gen, device="cuda", dtype=torch.float64) * hidden ** -0.5).to(dtype)
    dy = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64).to(dtype)
    return x, off, W1, W2, dy


def test_experts_gradients_against_differences(node):
    """In fp64: the derivative of <dy, y> along a random direction against central differences.  The function is of degree 3
    in W1 and smooth up to second order apart from relu's corner (the cube of it is smooth enough): with a step of 1e-5 the difference is off by about 1e-10 |third derivative|
    and the rounding by about 1e-16 / 1e-5 = 1e-11 of the value."""
    import torch
    x, off, W1, W2, dy = experts_case(torch.float64)
    gen = generator(12)
    dx, dW1, dW2 = (lambda e: (e.forward(x), e.backward(dy))[1])(Experts(node, off, W1, W2))
    for which, grad in enumerate((dx, dW1, dW2)):
        t = torch.randn(grad.shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        value = []
        for sign in (1, -1):
            at = [x, W1, W2]
            at[which] = at[which] + sign * h * t
            value.append(float((Experts(node, off, at[1], at[2]).forward(at[0]) * dy).sum()))
        slope, formula = (value[0] - value[1]) / (2 * h), float((grad * t).sum())
        assert abs(slope - formula) <= 1e-7 * float((grad * t).abs().sum()), (which, slope, formula)


@pytest.mark.parametrize("type_", ["bf16", "f16"])
def test_experts_gradients_against_the_formula(node, type_):
    """Every kernel's result against the 64-bit formula on the kernel's own (rounded) inputs is tested above; here the chain of four roundings
    to the type: each is half a step, and its effect passes through sums whose terms are independent: eight half steps of the norm are allowed."""
    import torch
    x, off, W1, W2, dy = experts_case(kind(type_), tokens=300, groups=5, d=136, hidden=200)
    e = Experts(node, off, W1, W2)
    y = e.forward(x)
    got = (y, *e.backward(dy))
    w = [t.double() for t in (x, W1, W2, dy)]
    want_y, want_dx, want_1, want_2 = torch.empty_like(w[0]), torch.empty_like(w[0]), torch.empty_like(w[1]), torch.empty_like(w[2])
    ends = off.tolist()
    for g, (a, b) in enumerate(zip(ends, ends[1:])):
        h = w[0][a:b] @ w[1][g].T
        act = h.relu().square()
        want_y[a:b] = act @ w[2][g].T
        da = w[3][a:b] @ w[2][g]
        dh = 2 * h.relu() * da
        want_2[g] = w[3][a:b].T @ act
        want_dx[a:b] = dh @ w[1][g]
        want_1[g] = dh.T @ w[0][a:b]
    for u, v in zip(got, (want_y, want_dx, want_1, want_2)):
        assert float((u.double() - v).norm() / v.norm()) <= 8 * torch.finfo(kind(type_)).eps / 2


def test_experts_in_a_graph_with_other_routings(node):
    """Captured once, replayed with other tokens and other group sizes in the same buffers: every replay equals the eager call."""
    import torch
    x, off, W1, W2, dy = experts_case(torch.bfloat16, tokens=200, groups=8, d=128, hidden=256)
    e = Experts(node, off, W1, W2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        e.forward(x); e.backward(dy)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = e.forward(x)
        grads = e.backward(dy)
    for seed in (21, 22, 23):
        gen = generator(seed)
        token, other = route(gen, 200, 8, 2)
        off.copy_(other)
        x.copy_(torch.randn(200, 128, generator=gen, device="cuda")[token])
        dy.copy_(torch.randn(dy.shape, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        eager = Experts(node, off, W1, W2)
        want = (eager.forward(x), *eager.backward(dy))
        assert all(torch.equal(a, b) for a, b in zip((y, *grads), want))


def test_experts_in_8_bits(node):
    """Weights and activations rounded to 8 bits: against the same steps in 64 bits on the kernel's own 8-bit numbers."""
    import torch
    x, off, W1, W2, _ = experts_case(torch.bfloat16, tokens=120, groups=6, d=256, hidden=320)

    def quantized(t):
        q, s = torch.empty(t.shape, dtype=torch.int8, device="cuda"), torch.empty(t.shape[:-1], device="cuda")
        assert node.quantize_i8_device(t.view(-1, t.shape[-1]), q.view(-1, t.shape[-1]), s.view(-1)) == 0
        return q, s

    (q1, s1), (qx, sx) = quantized(W1), quantized(x)
    h = torch.empty(x.shape[0], W1.shape[1], dtype=torch.bfloat16, device="cuda")
    assert node.grouped_gemm_i8_device(off, q1, s1, qx, sx, h) == 0
    ends = off.tolist()
    for g, (a, b) in enumerate(zip(ends, ends[1:])):
        assert torch.equal(h[a:b], scaled(qx[a:b].double() @ q1[g].double().T, s1[g], sx[a:b], torch.bfloat16))
        # each of the k products is off by at most half a step of either side, s / 2 times the other's magnitude, and both
        ref = x[a:b].double() @ W1[g].double().T
        half = sx[a:b, None].double() / 2 * W1[g].double().abs().sum(1)[None] + s1[g][None].double() / 2 * x[a:b].double().abs().sum(1)[:, None] \
            + 256 * sx[a:b, None].double() * s1[g][None].double() / 4
        assert bool(((h[a:b].double() - ref).abs() <= half * 1.01 + ref.abs() * 2 ** -8).all())


@pytest.mark.parametrize("type_", ["bf16", "f64"])
def test_gradients_without_scratch_memory(node, type_):
    """The C call with no scratch memory, with too little and with enough: all within the bound, equal calls equal bits."""
    import torch
    gen, k, m, n = generator(51), 20000, 200, 136
    X = torch.randn(k, m, generator=gen, device="cuda", dtype=torch.float64).to(kind(type_))
    Y = torch.randn(k, n, generator=gen, device="cuda", dtype=torch.float64).to(kind(type_))
    off = offsets_of([k - 70], 40)
    lib, code = node.lib.load(), {"bf16": node.AMD_BF16, "f64": node.AMD_F64}[type_]
    size = lib.starneig_amd_grouped_outer_work_size(code, 1, m, n, k)
    assert size > 0
    work = torch.full((size + 16,), 171, dtype=torch.uint8, device="cuda")
    x, y = X[40:k - 30].double(), Y[40:k - 30].double()
    ref, mag = y.T @ x, y.T.abs() @ x.abs()
    bound = product_bound(k, mag, ref, kind(type_))
    stream = torch.cuda.current_stream().cuda_stream
    for given in (0, 16, size - 16, size):
        got = []
        for _ in range(2):
            D = torch.full((1, n, m), float("nan"), dtype=kind(type_), device="cuda")
            assert lib.starneig_amd_grouped_outer_device(code, code, 1, m, n, k, off.data_ptr(), X.data_ptr(), m, Y.data_ptr(), n, 0.0,
                                                         D.data_ptr(), m, m * n, work.data_ptr() if given else None, given, stream) == 0
            got.append(D)
        assert torch.equal(got[0], got[1])
        assert bool(((got[0][0].double() - ref).abs() <= bound).all())
    assert bool((work[size:] == 171).all())


def test_two_gradients_at_once_in_a_graph(node):
    """Two long sums on two branches of one graph, each with scratch memory of its own: every replay equals the eager results."""
    import torch
    gen = generator(52)
    data = [(torch.randn(16000, 192, generator=gen, device="cuda").bfloat16(), torch.randn(16000, 128, generator=gen, device="cuda").bfloat16(),
             torch.zeros(1, 128, 192, device="cuda")) for _ in range(2)]
    off = offsets_of([16000])

    def both():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert node.grouped_outer_device(off, *data[1]) == 0
        assert node.grouped_outer_device(off, *data[0]) == 0
        torch.cuda.current_stream().wait_stream(side)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(4):
        for x, y, d in data:
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
            d.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for x, y, d in data:
            eager = torch.empty_like(d)
            assert node.grouped_outer_device(off, x, y, eager) == 0
            assert torch.equal(d, eager)


def test_equal_calls_give_equal_bits(node):
    import torch
    gen = generator(53)
    sizes, m, k = [700, 0, 3, 1500], 520, 712
    A = torch.randn(len(sizes), m, k, generator=gen, device="cuda").half()
    B = torch.randn(sum(sizes), k, generator=gen, device="cuda").half()
    off, seen = offsets_of(sizes), []
    for _ in range(5):
        C = torch.empty(sum(sizes), m, dtype=torch.float16, device="cuda")
        D = torch.empty(len(sizes), m, k, device="cuda")
        assert node.grouped_gemm_device("T", off, A, B, C) == 0
        assert node.grouped_outer_device(off, B, C, D) == 0
        seen.append((C, D))
    assert all(torch.equal(c, seen[0][0]) and torch.equal(d, seen[0][1]) for c, d in seen)


def test_infinities_and_nan_stay_in_their_columns(node):
    """A column that holds an infinity or a NaN spoils its own results and no others, also next to a group's end and in a cut last inner chunk."""
    import torch
    gen = generator(54)
    for k in (72, 203, 640):
        sizes = [65, 3, 130]
        n = sum(sizes)
        A = torch.randn(3, 96, k, generator=gen, device="cuda").bfloat16()
        B = torch.randn(n, k, generator=gen, device="cuda").bfloat16()
        clean = torch.empty(n, 96, dtype=torch.bfloat16, device="cuda")
        assert node.grouped_gemm_device("T", offsets_of(sizes), A, B, clean) == 0
        bad = [0, 64, 65, 67, n - 1]
        for i, c in enumerate(bad):
            B[c, (k - 1) * (i % 2)] = float("nan") if i % 3 else float("inf")
        C = torch.empty_like(clean)
        assert node.grouped_gemm_device("T", offsets_of(sizes), A, B, C) == 0
        fine = torch.ones(n, dtype=torch.bool, device="cuda")
        fine[bad] = False
        assert torch.equal(C[fine], clean[fine])
        assert not bool(C[~fine].isfinite().any())


def test_two_streams_at_once(node):
    import torch
    cases = [experts_case(torch.bfloat16, seed=s, tokens=400, groups=8, d=256, hidden=512) for s in (31, 32)]
    torch.cuda.synchronize()
    alone = []
    for x, off, W1, W2, dy in cases:
        e = Experts(node, off, W1, W2)
        alone.append((e.forward(x), *e.backward(dy)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i, (x, off, W1, W2, dy) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                e = Experts(node, off, W1, W2)
                got[i] = (e.forward(x), *e.backward(dy))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_far_offsets(node):
    """Columns and matrices whose positions pass 2^31 entries."""
    import torch
    n, k, m = 66000, 33000, 24
    B = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
    B[: n - 40].zero_()
    gen = generator(41)
    B[n - 40:] = torch.randn(40, k, generator=gen, device="cuda").bfloat16()
    A = torch.randn(1, m, k, generator=gen, device="cuda").bfloat16()
    C = torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
    assert node.grouped_gemm_device("T", offsets_of([n]), A, B, C) == 0
    ref, mag = B[n - 40:].double() @ A[0].double().T, B[n - 40:].double().abs() @ A[0].double().abs().T
    assert bool(((C[n - 40:].double() - ref).abs() <= product_bound(k, mag, ref, torch.bfloat16)).all())
    assert bool((C[: n - 40] == 0).all())
    Y = torch.randn(n, 8, generator=gen, device="cuda").bfloat16()
    D = torch.empty(1, 8, k, device="cuda")
    assert node.grouped_outer_device(offsets_of([40], n - 40), B, Y, D) == 0
    ref, mag = Y[n - 40:].double().T @ B[n - 40:].double(), Y[n - 40:].double().abs().T @ B[n - 40:].double().abs()
    assert bool(((D[0].double() - ref).abs() <= product_bound(40, mag, ref, torch.float32)).all())


def test_refusals_on_the_gpu(node):
    import torch
    off = offsets_of([2, 2])
    A = torch.zeros(2, 6, 8, dtype=torch.bfloat16, device="cuda")
    B, C = torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 6, dtype=torch.bfloat16, device="cuda")
    bad = [("T", off, A[:1], B, C), ("T", off, A, B, C.float()), ("T", off.long(), A, B, C), ("T", off, A, B.T, C), ("N", off, A, B, C),
           ("T", off, A.cpu(), B, C), ("T", off, A, B, C[:3]), ("T", off[:1], A, B, C), ("T", off, A.char(), B.char(), C.char())]
    for args in bad:
        with pytest.raises(ValueError):
            node.grouped_gemm_device(*args)
    f = torch.zeros(4, 8, device="cuda")
    assert node.grouped_gemm_device("T", off, A.float(), f, C.float()) == -1
    assert node.grouped_gemm_device("X", off, A.transpose(1, 2).contiguous(), B, C) == -2
    with pytest.raises(ValueError):
        node.gemm_i8_device(A[0].char(), torch.zeros(5, device="cuda"), B.char(), torch.zeros(4, device="cuda"), C)
    assert node.gemm_i8_device(A[0].char(), torch.zeros(6, device="cuda"), B.char(), torch.zeros(4, device="cuda"), C.double()) == -1


@pytest.mark.parametrize("type_", TYPES)
def test_the_most_groups(node, type_):
    """65535 groups, nearly all empty: the products of the few columns, and zeros or beta D from the others."""
    import torch
    gen, dtype, groups, m, n, k = generator(71), kind(type_), 65535, 24, 9, 40
    sizes = np.zeros(groups, dtype=int)
    filled = {0: 2, 63: 1, 64: 3, 40000: 17, groups - 1: 20}
    for g, size in filled.items():
        sizes[g] = size
    total = sum(filled.values())
    A = padded(gen, 1, m, k, dtype=dtype)
    B, C = padded(gen, total, k, dtype=dtype), padded(gen, total, m, dtype=dtype)
    assert node.grouped_gemm_device("T", offsets_of(sizes), A.expand(groups, m, k), B, C) == 0
    a, b = A[0].double().T, B.double()
    ref = b @ a
    assert bool(((C.double() - ref).abs() <= product_bound(k, b.abs() @ a.abs(), ref, dtype)).all())
    X, Y = padded(gen, total, m, dtype=dtype), padded(gen, total, n, dtype=dtype)
    D = torch.full((groups, n, m), 3.0, dtype=dtype, device="cuda")
    assert node.grouped_outer_device(offsets_of(sizes), X, Y, D, beta=0.5) == 0
    at = 0
    for g, size in filled.items():
        x, y = X[at:at + size].double(), Y[at:at + size].double()
        ref = y.T.contiguous() @ x + 1.5
        bound = product_bound(size + 2, y.abs().T.contiguous() @ x.abs() + 1.5, ref, dtype)
        assert bool(((D[g].double() - ref).abs() <= bound).all()), g
        at += size
    empty = torch.ones(groups, dtype=torch.bool, device="cuda")
    empty[list(filled)] = False
    assert bool((D[empty] == 1.5).all())


@pytest.mark.parametrize("tokens", [1, 50])
def test_8_bit_groups_that_share_their_scales(node, tokens):
    """One matrix and one row of scales for all groups (strides of zero), some groups without a column."""
    import torch
    gen, groups, m, k = generator(73), 5, 130, 264
    sizes = [0, tokens, 0, 2, tokens]
    n = sum(sizes)
    A, B = whole(gen, 1, m, k), whole(gen, n, k)
    sa, sb = torch.rand(1, m, generator=gen, device="cuda"), torch.rand(n, generator=gen, device="cuda")
    C = torch.empty(n, m, dtype=torch.float32, device="cuda")
    assert node.load().starneig_amd_grouped_gemm_i8_device(
        node.AMD_F32, groups, m, n, k, offsets_of(sizes).data_ptr(), A.data_ptr(), k, 0, sa.data_ptr(), 0, B.data_ptr(), k, sb.data_ptr(), C.data_ptr(), m,
        torch.cuda.current_stream().cuda_stream) == 0
    sums = B.double() @ A[0].double().T.contiguous()
    assert torch.equal(C, scaled(sums, sa[0], sb, torch.float32))


@pytest.mark.parametrize("trans", ["T", "N"])
def test_f64_columns_too_far_apart_for_direct_loads(node, trans):
    """Columns more than 4 MB apart are read by another kernel."""
    import torch
    gen, sizes, m, k, ld = generator(79), [300, 0, 500, 266], 330, 333, (1 << 19) + 3
    n = sum(sizes)
    far = torch.empty((n + 340, ld), dtype=torch.float64, device="cuda")
    far[:, :400] = float("nan")
    A = torch.randn(1, *((m, k) if trans == "T" else (k, m)), generator=gen, device="cuda", dtype=torch.float64)
    B = torch.randn(n, k, generator=gen, device="cuda", dtype=torch.float64)
    farA, farB = far[:A.shape[1], :A.shape[2]], far[340:, :k]
    farA.copy_(A[0]); farB.copy_(B)
    near, there = torch.empty(n, m, dtype=torch.float64, device="cuda"), torch.empty(n, m, dtype=torch.float64, device="cuda")
    off, groups = offsets_of(sizes), len(sizes)
    assert node.grouped_gemm_device(trans, off, A.expand(groups, *A.shape[1:]), B, near) == 0
    assert node.grouped_gemm_device(trans, off, farA[None].expand(groups, *A.shape[1:]), farB, there) == 0
    a = A[0].T if trans == "T" else A[0]
    ref = B @ a
    bound = product_bound(k, B.abs() @ a.abs(), ref, torch.float64)
    assert bool(((near - ref).abs() <= 2 * bound).all()) and bool(((there - ref).abs() <= 2 * bound).all())
    # and without inner terms
    assert node.grouped_gemm_device(trans, off, farA[None].expand(groups, *A.shape[1:])[:, :, :0] if trans == "T" else
                                    farA[None].expand(groups, *A.shape[1:])[:, :0], farB[:, :0], there) == 0
    assert bool((there == 0).all())
    Y = torch.randn(n, 40, generator=gen, device="cuda", dtype=torch.float64)
    for beta in (0.0, 0.5):
        D = torch.ones(groups, 40, k, dtype=torch.float64, device="cuda")
        E = D.clone()
        assert node.grouped_outer_device(off, B, Y, D, beta=beta) == 0
        assert node.grouped_outer_device(off, farB, Y, E, beta=beta) == 0
        bound = product_bound(max(sizes) + 2, torch.stack([y.abs().T.contiguous() @ x.abs() for y, x in zip(Y.split(sizes), B.split(sizes))]) + beta, D, torch.float64)
        assert bool(((D - E).abs() <= 2 * bound).all())


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("k", [1, 2, 3, 15, 16, 17, 31, 33, 48, 257, 300])
@pytest.mark.parametrize("pads,shifts", [((0, 0, 0), (0, 0, 0)), ((1, 3, 5), (1, 0, 3))])
def test_f64_tiles(node, trans, k, pads, shifts):
    """Enough tiles for those of 64 x 64, inner lengths around theirs of 16."""
    check_product(node, trans, "f64", [300, 0, 450, 1, 64], 701, k, first=2, behind=3, pads=pads, shifts=shifts, seed=83)


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("k", [1, 7, 8, 9, 63, 64, 65, 500, 519])
@pytest.mark.parametrize("pads,shifts", [((0, 0, 0), (0, 0, 0)), ((1, 3, 5), (1, 0, 3))])
def test_f64_of_few_columns(node, trans, k, pads, shifts):
    """Few outputs: 16 columns a workgroup, whose waves cut inner lengths around multiples of 8 and 64."""
    check_product(node, trans, "f64", [3, 0, 17, 40], 50, k, first=2, behind=3, pads=pads, shifts=shifts, seed=89)


@pytest.mark.parametrize("type_,out", [("bf16", "f32"), ("f16", "f16"), ("f64", "f64")])
@pytest.mark.parametrize("beta", [0.0, 0.5])
@pytest.mark.parametrize("k,m,n", [(4203, 64, 64), (2118, 70, 9), (9000, 33, 130), (700, 64, 64)])
def test_outer_of_long_sums(node, type_, out, beta, k, m, n):
    """Few outputs, many slices, whose sums several threads add up."""
    check_outer(node, type_, out, [k], m, n, beta, pads=(0, 2, 1), shifts=(0, 0, 0), seed=97)


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("k", [1, 17, 32, 63, 270])
@pytest.mark.parametrize("pads,shifts", [((0, 0, 0), (0, 0, 0)), ((1, 3, 5), (1, 0, 3))])
def test_f64_of_many_tiles(node, trans, k, pads, shifts):
    """More tiles than the chip holds at once."""
    check_product(node, trans, "f64", [3000, 0, 1, 700], 701, k, first=2, behind=3, pads=pads, shifts=shifts, seed=101)
