"""Argument checks of the fp8 and dropout entry points, and the restatement the
GPU tests compare with.  No GPU."""
import pytest
import torch

import _fp8_ref as ref
from test_philox_gpu import philox_py


def test_python_refusals():
    import advanced_optimizers_b200 as A
    x = torch.zeros(4, 256)
    with pytest.raises(NotImplementedError, match="CUDA device"):
        A.philox_dropout(x, 0.1)
    with pytest.raises(NotImplementedError, match="CUDA device"):
        A.quantize_fp8(x)
    with pytest.raises(NotImplementedError, match="CUDA device"):
        A.fp8_linear(x, torch.zeros(8, 256))
    with pytest.raises(NotImplementedError, match="blocks of"):
        A.quantize_fp8(x, (1, 64))
    with pytest.raises(NotImplementedError, match="codes are"):
        A.quantize_fp8(x, dtype=torch.int8)
    with pytest.raises(ValueError, match="layout"):
        A.quantize_fp8(x, layout="columns")
    with pytest.raises(ValueError, match="matrix"):
        A.quantize_fp8(x[0])
    with pytest.raises(ValueError, match=r"\[\.\.\., K\]"):
        A.fp8_linear(x, torch.zeros(8, 255))
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    with pytest.raises(NotImplementedError, match="codes are"):
        A.Fp8Blocks(x, torch.zeros(4, 2))
    with pytest.raises(NotImplementedError, match="CUDA device"):
        A.Fp8Blocks(x.to(e4), torch.ones(4, 2).to(e8))


@pytest.mark.parametrize("bad", [dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(seed=-1), dict(seed=1 << 64), dict(site=1 << 32),
                                 dict(step=-1), dict(step=1 << 32), dict(step=torch.zeros(2, dtype=torch.int64)),
                                 dict(step=torch.zeros(1, dtype=torch.int32))])
def test_dropout_arguments(bad):
    from advanced_optimizers_b200.dropout import drop_fields
    kw = {**dict(p=0.1, seed=1, site=0, step=0, device=torch.device("cpu")), **bad}
    with pytest.raises(ValueError):
        drop_fields(**kw)


def test_dropout_threshold_and_scale():
    from advanced_optimizers_b200.dropout import drop_fields
    for p, T in ((0.0, 0), (1e-6, 0), (0.5, 32768), (0.1, 6554), (1.0, 65536)):
        *_, threshold, scale = drop_fields(p, 1, 0, 0, None)
        assert threshold == T and scale == (65536 / (65536 - T) if T < 65536 else 0.0)


def test_packed_structs_match_the_header():
    from advanced_optimizers_b200 import _lib as L
    from advanced_optimizers_b200 import dropout, fp8
    lib = L.lib()
    for which, s in ((10, dropout.SPEC), (11, fp8._QUANT), (12, fp8._GEMM)):
        assert lib.advopt_sizeof(which) == s.size


def quant_args(**kw):
    from advanced_optimizers_b200 import fp8
    f = dict(x=4096, ldx=256, rows=4, cols=256, codes_r=8192, ld_r=256, scales_r=16384, ld_sr=4, codes_c=0, ld_c=0, scales_c=0,
             ld_sc=0, partial=0, x_dtype=1, tile=0, code=0, pad=0, seed=1, step_dev=0, site=0, step=0, threshold=0, scale=1.0)
    f.update(kw)
    return fp8._QUANT.pack(*f.values())


@pytest.mark.parametrize("bad", [dict(x=0), dict(ldx=255), dict(rows=-1), dict(cols=-1), dict(x_dtype=2), dict(code=2), dict(tile=2),
                                 dict(codes_r=0), dict(scales_r=0), dict(ld_r=248), dict(ld_r=240), dict(codes_r=8200), dict(ld_sr=1),
                                 dict(codes_c=8192, ld_c=16, scales_c=0), dict(codes_c=8192, ld_c=8, scales_c=4096, ld_sc=1),
                                 dict(codes_c=8192, ld_c=16, scales_c=4096, ld_sc=0), dict(threshold=65537), dict(step_dev=4),
                                 dict(rows=1 << 38)])
def test_quantize_c_refusals(bad):
    from advanced_optimizers_b200 import _lib as L
    assert L.lib().advopt_fp8_quantize(quant_args(**bad), None) in (-1, -3)
    assert L.lib().advopt_last_error()
    assert L.lib().advopt_fp8_quantize(None, None) == -1


def gemm_args(**kw):
    from advanced_optimizers_b200 import fp8
    f = dict(a=4096, lda=256, sa=1024, ldsa=4, b=8192, ldb=256, sb=2048, ldsb=4, d=65536, ldd=128, bias=0, residual=0, ldres=128,
             m=4, n=128, k=256, a_code=0, b_code=0, a_tile=0, b_tile=0, d_dtype=1, variant=0, err=0, seed=1, step_dev=0, site=0,
             step=0, threshold=0, scale=1.0)
    f.update(kw)
    return fp8._GEMM.pack(*f.values())


@pytest.mark.parametrize("bad", [dict(a=0), dict(b=0), dict(sa=0), dict(sb=0), dict(d=0), dict(m=-1), dict(n=-1), dict(k=0),
                                 dict(d_dtype=2), dict(a_code=2), dict(b_code=-1), dict(a=4104), dict(b=8200), dict(lda=248),
                                 dict(ldb=240), dict(sa=1026), dict(ldsa=2), dict(ldsb=0), dict(sb=2049), dict(ldd=127),
                                 dict(residual=4096, ldres=100), dict(threshold=1 << 20), dict(step_dev=1), dict(m=1 << 31),
                                 dict(n=1 << 31, ldd=1 << 31), dict(variant=160),
                                 dict(variant=-1), dict(variant=100256), dict(variant=3128), dict(variant=8032), dict(variant=201128)])
def test_gemm_c_refusals(bad):
    from advanced_optimizers_b200 import _lib as L
    assert L.lib().advopt_fp8_gemm(gemm_args(**bad), None) in (-1, -3)
    assert L.lib().advopt_last_error()
    assert L.lib().advopt_fp8_gemm(None, None) == -1


def test_dropout_and_col_sum_c_refusals():
    from advanced_optimizers_b200 import _lib as L
    from advanced_optimizers_b200.dropout import SPEC
    ok = SPEC.pack(1, 0, 0, 0, 100, 1.0)
    lib = L.lib()
    assert lib.advopt_dropout(None, None, None, 5, 0, ok, None) == -1
    assert lib.advopt_dropout(4096, 4096, None, -1, 0, ok, None) == -1
    assert lib.advopt_dropout(4096, 4096, None, 5, 0, None, None) == -1
    assert lib.advopt_dropout(4096, 4096, None, 5, 2, ok, None) == -3
    assert lib.advopt_dropout(4096, 4096, None, 5, 0, SPEC.pack(1, 0, 0, 0, 65537, 1.0), None) == -1
    assert lib.advopt_dropout(None, None, None, 0, 0, ok, None) == 0
    assert lib.advopt_col_sum(None, None, 1, 5, 0, None) == -1
    assert lib.advopt_col_sum(4096, None, 1, 5, 0, None) == -1
    assert lib.advopt_col_sum(4096, 4096, 1, 5, 3, None) == -3
    assert lib.advopt_col_sum(None, None, 0, 0, 0, None) == 0


def test_restated_mask_is_philox():
    r = ref.random16(40, (5 << 32) | 9, 3, 17, first=13)
    for i in range(40):
        k = 13 + i
        w = philox_py([k >> 3, 4 << 24, 3, 17], [9, 5])
        assert int(r[i]) == (w[(k & 7) >> 1] >> (16 * (k & 1))) & 0xFFFF


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_restated_codes_are_the_types_values(dtype):
    """The restatement's codes are numbers of the type, nearest to what they stand for, and its scales the least that fit."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(9, 300, generator=g) * torch.exp2(torch.randint(-20, 20, (9, 1), generator=g).float())
    for block in (1, 128):
        q, e = ref.quantize(x, block, dtype)
        assert torch.equal(q, q.to(torch.float32).to(dtype).to(torch.float64))
        scaled = x.double() / ref.blocked(ref.pow2(e), 9, 300, block)
        assert torch.equal(q.float(), scaled.float().to(dtype).float())
        top = scaled.abs().max()
        assert float(top) <= ref.LARGEST[dtype]
        assert float(2 * scaled.abs().amax()) > ref.LARGEST[dtype]


