"""GPU: positions that pass 2^31 entries, in each operand of each product, and the 8-bit calls and long fp64 sums in captured graphs.
Bounds as in test_gpu_products.py."""
import pytest

from test_gpu_products import generator, offsets_of, product_bound, route, scaled, whole

pytestmark = pytest.mark.gpu


def test_far_columns_in_8_bits(node):
    """The rounding of columns behind 2^31 numbers, and their product."""
    import torch
    n, k, m, last = 66000, 33000, 24, 40
    gen = generator(41)
    X = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    X[n - last:] = torch.randn(last, k, generator=gen, device="cuda").bfloat16()
    Q, scale = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    assert node.quantize_i8_device(X, Q, scale) == 0
    near, near_scale = torch.empty(last, k, dtype=torch.int8, device="cuda"), torch.empty(last, device="cuda")
    assert node.quantize_i8_device(X[n - last:].clone(), near, near_scale) == 0
    assert torch.equal(Q[n - last:], near) and torch.equal(scale[n - last:], near_scale) and bool((scale[:n - last] == 0).all()) and not bool(Q[:n - last].any())
    A, sa = whole(gen, 1, m, k), torch.rand(1, m, generator=gen, device="cuda")
    C = torch.empty(n, m, device="cuda")
    assert node.grouped_gemm_i8_device(offsets_of([n]), A, sa, Q, scale, C) == 0
    assert torch.equal(C[n - last:], scaled(near.double() @ A[0].double().T.contiguous(), sa[0], near_scale, torch.float32)) and not bool(C[:n - last].any())


@pytest.mark.parametrize("trans", ["T", "N"])
@pytest.mark.parametrize("type_,groups,columns", [("bf16", 2100, 9), ("bf16", 2100, 3000), ("f64", 2100, 9), ("f64", 2100, 20000)])
def test_far_matrices(node, trans, type_, groups, columns):
    """A group whose matrix lies behind 2^31 numbers, by the kernels of few columns and of many."""
    import torch
    dtype, m, k = {"bf16": torch.bfloat16, "f64": torch.float64}[type_], 1024, 1032
    gen, sizes = generator(43), [0] * groups
    sizes[groups - 2], sizes[3] = columns, 5
    A = torch.empty(groups, *((m, k) if trans == "T" else (k, m)), dtype=dtype, device="cuda")
    for g in (3, groups - 2):
        A[g] = torch.randn(A.shape[1:], generator=gen, device="cuda")
    B = torch.randn(columns + 5, k, generator=gen, device="cuda").to(dtype)
    C = torch.empty(columns + 5, m, dtype=dtype, device="cuda")
    assert node.grouped_gemm_device(trans, offsets_of(sizes), A, B, C) == 0
    for g, at, end in ((3, 0, 5), (groups - 2, 5, columns + 5)):
        a, b = (A[g].double().T if trans == "T" else A[g].double()).contiguous(), B[at:end].double()
        ref = b @ a
        assert bool(((C[at:end].double() - ref).abs() <= product_bound(k, b.abs() @ a.abs(), ref, dtype)).all()), g


@pytest.mark.parametrize("type_,out", [("bf16", "f32"), ("f64", "f64")])
def test_far_gradients(node, type_, out):
    """Gradients that lie behind 2^31 numbers, others that have no column, beta."""
    import torch
    kinds = {"bf16": torch.bfloat16, "f32": torch.float32, "f64": torch.float64}
    groups, m, n, columns = 2100, 1024, 1032, 300
    gen, sizes = generator(47), [0] * groups
    sizes[groups - 2] = columns
    X, Y = (torch.randn(columns, s, generator=gen, device="cuda").to(kinds[type_]) for s in (m, n))
    D = torch.ones(groups, n, m, dtype=kinds[out], device="cuda")
    assert node.grouped_outer_device(offsets_of(sizes), X, Y, D, beta=0.5) == 0
    x, y = X.double(), Y.double().T.contiguous()
    ref = y @ x + 0.5
    assert bool(((D[groups - 2].double() - ref).abs() <= product_bound(columns + 2, y.abs() @ x.abs() + 0.5, ref, kinds[out])).all())
    assert bool((D[:groups - 2] == 0.5).all()) and bool((D[groups - 1] == 0.5).all())


def test_8_bit_products_in_a_graph(node):
    """Rounding and product, captured once and replayed with other columns and other groups, with eager calls in between."""
    import torch
    gen, tokens, groups, m, k = generator(53), 200, 8, 264, 520
    A, sa = whole(gen, groups, m, k), torch.rand(groups, m, generator=gen, device="cuda")
    n = tokens * 2
    x, off = torch.empty(n, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    q, s, C = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, m, device="cuda")

    def step(q, s, C):
        assert node.quantize_i8_device(x, q, s) == 0
        assert node.grouped_gemm_i8_device(off, A, sa, q, s, C) == 0

    x.zero_()
    step(q, s, C)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, s, C)
    for _ in range(4):
        token, other = route(gen, tokens, groups, 2)
        off.copy_(other)
        x.copy_(torch.randn(tokens, k, generator=gen, device="cuda")[token])
        C.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(t) for t in (q, s, C)]
        step(*eager)
        assert all(torch.equal(a, b) for a, b in zip((q, s, C), eager))


def test_long_f64_sums_in_a_graph(node):
    import torch
    gen, k, m, n = generator(59), 9000, 70, 40
    X, Y, D = torch.empty(k, m, dtype=torch.float64, device="cuda"), torch.empty(k, n, dtype=torch.float64, device="cuda"), torch.zeros(2, n, m, dtype=torch.float64, device="cuda")
    off = offsets_of([4000, 5000])
    assert node.lib.load().starneig_amd_grouped_outer_work_size(node.AMD_F64, 2, m, n, k) > 0
    X.zero_(); Y.zero_()
    assert node.grouped_outer_device(off, X, Y, D, beta=0.5) == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert node.grouped_outer_device(off, X, Y, D, beta=0.5) == 0
    for _ in range(4):
        X.normal_(generator=gen); Y.normal_(generator=gen); D.normal_(generator=gen)
        eager = D.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert node.grouped_outer_device(off, X, Y, eager, beta=0.5) == 0
        assert torch.equal(D, eager)
