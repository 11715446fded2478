"""A linear product's result may be written over its residual, but not over its input: every tile of
columns reads the input's whole rows."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["mixed", "fp32"])
@pytest.mark.parametrize("rows,cols", [(1, 40), (300, 640), (3, 65)])
def test_the_input_is_no_place_for_the_result(mode, rows, cols):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(B.param_dtype(mode))
    w = torch.randn(cols, cols, generator=g, device="cuda").to(x.dtype).float()
    b = torch.randn(cols, generator=g, device="cuda").to(x.dtype).float()
    before = x.clone()
    with B.store_of([w, b], mode) as store:
        for call in (lambda **k: store.linear(1, x, **k), lambda **k: store.linear(1, x, bias=2, **k),
                     lambda **k: store.linear_input_grad(1, x, add=k.pop("residual", None), **k)):
            for k in (dict(out=x), dict(residual=x, out=x)):
                with pytest.raises(ValueError, match="overlap"):
                    call(**k)
        assert torch.equal(x, before)
        # the input as the residual, and the residual's place, stay allowed
        want = store.linear(1, x, residual=x)
        res = x.clone()
        assert torch.equal(store.linear(1, x, residual=res, out=res), want)
        assert torch.equal(x, before)
        # a single row in the place of the bias that it reads
        bias = store.tensors[2].torch_view().view(1, cols)
        with pytest.raises(ValueError, match="overlap"):
            store.linear(1, x[:1], bias=2, residual=bias, out=bias)
        assert torch.equal(bias[0].float(), b)
