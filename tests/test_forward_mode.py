"""Forward-mode derivatives through the 8-bit products and the norms: there are none, and a call that is asked for one says
so.  The tangents are looked for before anything else, so this runs without a GPU."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw


def _weight(n=5, k=256):
    from engraft_ngram_amd import fp8
    return fp8.Fp8Weight(torch.zeros((n, k), dtype=torch.uint8).view(torch.float8_e4m3fn),
                         torch.zeros((1, 4), dtype=torch.uint8).view(torch.float8_e8m0fnu), k)


def _calls():
    from engraft_ngram_amd import fp8, norm
    w, one = _weight(), torch.ones(256)
    return {
        "product": lambda x: fp8.product(x, w),
        "product_lead": lambda x: fp8.product(x.reshape(3, 1, 256), w),
        "rms_norm": lambda x: norm.rms_norm(x),
        "rms_norm_weight": lambda x: norm.rms_norm(torch.zeros((3, 256)), x[0]),
        "add_rms_norm": lambda x: norm.add_rms_norm(x, torch.zeros((3, 256)), one),
        "add_rms_norm_residual": lambda x: norm.add_rms_norm(torch.zeros((3, 256)), x, one),
        "add_rms_norm_fp8": lambda x: norm.add_rms_norm(torch.zeros((3, 256)), x, one, out_dtype="fp8"),
        "normed_product": lambda x: norm.normed_product(x, None, one, w),
        "normed_product_residual": lambda x: norm.normed_product(torch.zeros((3, 256)), x, one, w),
    }


NAMES = ["product", "product_lead", "rms_norm", "rms_norm_weight", "add_rms_norm", "add_rms_norm_residual", "add_rms_norm_fp8",
         "normed_product", "normed_product_residual"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_not_dropped(name, grad):
    call = _calls()[name]
    with fw.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(fw.make_dual(torch.ones((3, 256)), torch.ones((3, 256))))
        # without a tangent, or where none is wanted, the call goes on (to the host tensors' refusal)
        with pytest.raises(ValueError, match="GPU"):
            call(torch.ones((3, 256)))
        with fw._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="GPU"):
            call(fw.make_dual(torch.ones((3, 256)), torch.ones((3, 256))))


def test_what_has_no_derivative_takes_the_values():
    """The calls without autograd treat a tangent as they treat requires_grad."""
    from engraft_ngram_amd import fp8, norm
    with fw.dual_level():
        x = fw.make_dual(torch.ones((3, 256)), torch.ones((3, 256)))
        for call in (lambda: fp8.quantize_rows(x), lambda: norm.add_rms_norm_stats(x, None, None),
                     lambda: norm.add_rms_norm_grad(x, x, torch.ones(3), None)):
            with pytest.raises(ValueError, match="GPU"):
                call()
