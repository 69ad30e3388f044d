"""The operators beside autograd: what they write in place, and what they do not record."""

import pytest
import torch


@pytest.mark.gpu
def test_what_is_written_in_place_is_known_to_autograd(native_lib):
    """A backward pass that saved a tensor before a call changed it fails, as after an operation of torch."""
    from leo_b200.gated_scan import gated_step
    from leo_b200.logits import adjust_logits

    def wide():
        return torch.randn(3, 8, device="cuda")

    x, w = wide(), wide().requires_grad_()
    state, base, logits, out, view = wide(), wide(), wide(), wide(), wide()
    for saved, call in ((state, lambda: gated_step(x, x, state)),
                        (base, lambda: gated_step(x[:, :4], x[:, :4], base[:, 2:6])),  # a view of what was saved
                        (logits, lambda: adjust_logits(logits, out=logits)),
                        (out, lambda: adjust_logits(x, out=out)),
                        (view, lambda: adjust_logits(x[:, :4], out=view[:, 4:]))):
        product = (saved * w).sum()
        before = saved._version
        call()
        assert saved._version > before
        with pytest.raises(RuntimeError, match="inplace"):
            product.backward()
    # reading changes nothing
    product = (x * w).sum()
    gated_step(x, x, state)
    adjust_logits(x)
    product.backward()
    assert torch.equal(w.grad, x)
    with torch.inference_mode():  # such tensors have no version
        lane = wide()
        gated_step(x, x, lane)
        adjust_logits(lane, out=lane)
