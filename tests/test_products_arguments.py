"""CPU: the grouped and 8-bit products refuse what they cannot do, argument by argument, before any GPU is touched."""
import pytest

import starneig_amd as S

P = 1 << 20             # any aligned address: nothing reads it, every call below ends at its checks


def call(name, args, **change):
    values = dict(args)
    assert set(change) <= set(values)
    values.update(change)
    return getattr(S.lib.load(), "starneig_amd_" + name)(*values.values())


GEMM = dict(type=S.AMD_BF16, trans=b"T", groups=2, m=8, n=6, k=16, off=P, A=P, ldA=16, strideA=128, B=P, ldB=16, C=P, ldC=8, stream=None)
OUTER = dict(type=S.AMD_F16, typeD=S.AMD_F32, groups=2, m=8, n=6, k=16, off=P, X=P, ldX=8, Y=P, ldY=6, beta=0.0, D=P, ldD=8, strideD=48, work=None, workSize=0, stream=None)
QUANT = dict(type=S.AMD_F32, k=16, n=3, X=P, ldX=16, Q=P, ldQ=16, scale=P, stream=None)
I8 = dict(typeC=S.AMD_BF16, m=8, n=6, k=16, A=P, ldA=16, sA=P, B=P, ldB=16, sB=P, C=P, ldC=8, stream=None)
GI8 = dict(typeC=S.AMD_F16, groups=2, m=8, n=6, k=16, off=P, A=P, ldA=16, strideA=128, sA=P, strideS=8, B=P, ldB=16, sB=P, C=P, ldC=8, stream=None)

BIG = (1 << 30) + 1

REFUSED = [
    ("grouped_gemm_device", GEMM, [
        (1, dict(type=S.AMD_F32)), (1, dict(type=7)), (1, dict(type=-1)), (2, dict(trans=b"C")), (3, dict(groups=0)), (3, dict(groups=65536)), (4, dict(m=-1)), (5, dict(n=-1)),
        (6, dict(k=-1)), (4, dict(m=BIG)), (5, dict(n=BIG)), (6, dict(k=BIG)), (7, dict(off=None)), (7, dict(off=P + 2)), (8, dict(A=None)), (8, dict(A=P + 1)), (9, dict(ldA=15)), (9, dict(trans=b"N", ldA=7)),
        (10, dict(strideA=-1)), (11, dict(B=None)), (11, dict(B=P + 1)), (12, dict(ldB=15)), (13, dict(C=None)), (13, dict(C=P + 1)), (14, dict(ldC=7))]),
    ("grouped_outer_device", OUTER, [
        (1, dict(type=S.AMD_F32)), (2, dict(typeD=S.AMD_BF16)), (2, dict(typeD=S.AMD_F64)), (2, dict(type=S.AMD_F64)), (3, dict(groups=0)), (4, dict(m=-1)),
        (5, dict(n=-1)), (6, dict(k=-1)), (4, dict(m=BIG)), (5, dict(n=BIG)), (6, dict(k=BIG)), (7, dict(off=None)), (8, dict(X=None)), (9, dict(ldX=7)), (10, dict(Y=None)), (11, dict(ldY=5)),
        (13, dict(D=None)), (13, dict(D=P + 2)), (14, dict(ldD=7)), (3, dict(groups=65536)), (15, dict(strideD=47)), (15, dict(strideD=0)), (16, dict(work=P + 8)), (17, dict(work=P, workSize=-1))]),
    ("quantize_i8_device", QUANT, [
        (1, dict(type=S.AMD_F64)), (1, dict(type=4)), (2, dict(k=-1)), (3, dict(n=-1)), (2, dict(k=BIG)), (3, dict(n=BIG)), (4, dict(X=None)), (4, dict(X=P + 2)), (5, dict(ldX=15)),
        (6, dict(Q=None)), (7, dict(ldQ=15)), (8, dict(scale=None)), (8, dict(scale=P + 1))]),
    ("gemm_i8_device", I8, [
        (1, dict(typeC=S.AMD_F64)), (2, dict(m=-1)), (3, dict(n=-1)), (2, dict(m=BIG)), (3, dict(n=BIG)), (4, dict(k=-1)), (4, dict(k=131072, ldA=131072, ldB=131072)), (5, dict(A=None)), (6, dict(ldA=15)),
        (7, dict(sA=None)), (7, dict(sA=P + 1)), (8, dict(B=None)), (9, dict(ldB=15)), (10, dict(sB=None)), (11, dict(C=None)), (11, dict(C=P + 1)), (12, dict(ldC=7))]),
    ("grouped_gemm_i8_device", GI8, [
        (1, dict(typeC=S.AMD_F64)), (2, dict(groups=0)), (2, dict(groups=65536)), (3, dict(m=-1)), (4, dict(n=-1)), (3, dict(m=BIG)), (4, dict(n=BIG)), (5, dict(k=-1)), (5, dict(k=131072, ldA=131072, ldB=131072)), (6, dict(off=None)), (7, dict(A=None)),
        (8, dict(ldA=15)), (9, dict(strideA=-1)), (10, dict(sA=None)), (11, dict(strideS=-1)), (12, dict(B=None)), (13, dict(ldB=15)), (14, dict(sB=None)),
        (15, dict(C=None)), (15, dict(C=P + 1)), (16, dict(ldC=7))]),
]


@pytest.mark.parametrize("name,args,position,change", [(n, a, p, c) for n, a, cs in REFUSED for p, c in cs])
def test_refused(name, args, position, change):
    assert call(name, args, **change) == -position


@pytest.mark.parametrize("name,args", [(n, a) for n, a, _ in REFUSED])
def test_not_initialised(name, args):
    assert not S.node_initialized()
    assert call(name, args) == S.NOT_INITIALIZED


def test_empty_sizes_need_no_pointers():
    assert call("grouped_gemm_device", GEMM, n=0, off=None, A=None, B=None, C=None) == S.NOT_INITIALIZED
    assert call("grouped_outer_device", OUTER, k=0, X=None, Y=None) == S.NOT_INITIALIZED
    assert call("grouped_outer_device", OUTER, groups=1, strideD=0) == S.NOT_INITIALIZED
    assert call("gemm_i8_device", I8, m=0, ldC=1, A=None, sA=None, B=None, sB=None, C=None) == S.NOT_INITIALIZED
    assert call("quantize_i8_device", QUANT, n=0, X=None, Q=None, scale=None) == S.NOT_INITIALIZED


def test_binding_refuses_host_tensors_and_shapes():
    import torch
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        S.grouped_gemm_device("T", off, torch.zeros(2, 6, 8, dtype=torch.bfloat16), x, torch.zeros(4, 6, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        S.grouped_gemm_device("T", off[:1], x, x, x)
    with pytest.raises(ValueError):
        S.quantize_i8_device(x, torch.zeros(4, 7, dtype=torch.int8), torch.zeros(4))


def test_work_size():
    size = S.lib.load().starneig_amd_grouped_outer_work_size
    assert size(S.AMD_BF16, 1, 512, 384, 20000) % (512 * 384 * 4) == 0 and size(S.AMD_BF16, 1, 512, 384, 20000) > 0      # few outputs, a long sum
    assert size(S.AMD_F16, 16, 4096, 2048, 32768) == 0              # outputs enough
    assert size(S.AMD_F64, 1, 512, 384, 20000) % (512 * 384 * 8) == 0 and size(S.AMD_F64, 1, 512, 384, 20000) > 0
    assert size(S.AMD_F64, 24, 312, 312, 40000) == 0
    for refused in [(S.AMD_F32, 1, 512, 384, 20000), (9, 1, 512, 384, 20000), (S.AMD_BF16, 0, 512, 384, 20000), (S.AMD_BF16, 65536, 512, 384, 20000),
                    (S.AMD_BF16, 1, 0, 384, 20000), (S.AMD_BF16, 1, 512, -1, 20000), (S.AMD_BF16, 1, 512, 384, 0)]:
        assert size(*refused) == 0
