"""advopt_dropout with the result in the input's or the residual's memory, as its contract allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,first", [(1, 0), (1003, 0), (1003, 1), (4096, 0), (3 << 20, 0), ((3 << 20) + 5, 0), (1 << 20, 3)])
def test_in_place_is_the_same(n, first, dtype):
    import advanced_optimizers_b200 as A
    from advanced_optimizers_b200 import _lib as L
    from advanced_optimizers_b200._device import dtype_code
    from advanced_optimizers_b200.dropout import SPEC, drop_fields
    key = dict(seed=11, site=2, step=5)
    g = torch.Generator(device="cuda").manual_seed(n)
    x, r = (torch.randn(n + first, generator=g, device="cuda").to(dtype)[first:] for _ in range(2))
    want, with_r = A.philox_dropout(x, 0.3, **key), A.philox_dropout(x, 0.3, residual=r, **key)
    spec = SPEC.pack(*drop_fields(0.3, 11, 2, 5, x.device))

    def call(y, x, r):
        L.check(L.lib().advopt_dropout(y.data_ptr(), x.data_ptr(), 0 if r is None else r.data_ptr(), n, dtype_code(dtype), spec,
                                       torch.cuda.current_stream().cuda_stream), "advopt_dropout")
        return y

    a = x.clone()
    assert torch.equal(call(a, a, None), want)
    a = x.clone()
    assert torch.equal(call(a, a, r), with_r)
    b = r.clone()
    assert torch.equal(call(b, x, b), with_r)
    both = x.clone()
    assert torch.equal(call(both, both, both), A.philox_dropout(x, 0.3, residual=x, **key))
