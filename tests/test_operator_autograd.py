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


@pytest.mark.gpu
def test_tangents_are_refused(native_lib):
    """Forward-mode differentiation: no call carries a tangent on, so none takes one; others go on as ever."""
    from torch.autograd import forward_ad

    from leo_b200.gated_scan import StoryLayout, gated_scan, gated_scan_backward, gated_step
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols

    x, h0 = torch.randn(5, 8, device="cuda"), torch.randn(2, 8, device="cuda")
    bias, ones, target = torch.randn(8, device="cuda"), torch.ones(5, device="cuda"), torch.ones(5, device="cuda").int()
    layout = StoryLayout([0, 2, 5], "cuda:0")
    carries = gated_scan(x, x, layout, keep_carries=True).carries
    with forward_ad.dual_level():
        dual, dual_h0 = (forward_ad.make_dual(v, torch.ones_like(v)) for v in (x, h0))
        dual_bias, dual_ones = (forward_ad.make_dual(v, torch.ones_like(v)) for v in (bias, ones))
        for call in (lambda: gated_scan(dual, x, layout), lambda: gated_scan(x, dual, layout),
                     lambda: gated_scan(x, x, layout, dual_h0),
                     lambda: gated_scan_backward(dual, x, x, layout, carries),
                     lambda: gated_scan_backward(x, x, x, layout, carries, grad_final=dual_h0),
                     lambda: gated_step(dual, x, x.clone()), lambda: gated_step(x, x, dual),
                     lambda: adjust_logits(dual), lambda: adjust_logits(x, bias=dual_bias),
                     lambda: adjust_logits(x, repetition=dual_ones), lambda: adjust_logits(x, out=dual),
                     lambda: pick_symbols(dual), lambda: masked_cross_entropy(dual, target),
                     lambda: masked_cross_entropy(x, target, weights=dual_ones)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        inside = (gated_scan(x, x, layout, h0).states, adjust_logits(x, bias=bias))
        with torch.no_grad():  # which does not stop tangents
            with pytest.raises(ValueError, match="tangent"):
                gated_scan(dual, x, layout)
    assert torch.equal(inside[0], gated_scan(x, x, layout, h0).states)
    assert torch.equal(inside[1], adjust_logits(x, bias=bias))
