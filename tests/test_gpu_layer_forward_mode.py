"""Forward-mode differentiation is not provided by the layer's operators: a tangent is refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from test_gpu_layer_ops import randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nsa():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nsa_from_scratch_b200 as m
    return m


def test_tangents_are_refused(nsa):
    x, w, sq, v = randn(8, 64, seed=1), randn(64, seed=2), randn(64, 64, seed=3), randn(64, 64, seed=4)
    e, es = nsa.quantize_rows_to_fp8(x)
    k, ks = nsa.quantize_rows_to_fp8(sq)
    q, pos, inv = randn(1, 8, 2, 64, seed=5), torch.arange(8, device="cuda").view(1, 1, 8), nsa.rope_frequencies(64)
    t = torch.ones_like
    dual = fwad.make_dual
    calls = [
        lambda: nsa.rms_norm(dual(x, t(x)), w), lambda: nsa.rms_norm(x, dual(w, t(w))), lambda: nsa.rms_norm(x, w, residual=dual(x, t(x))),
        lambda: nsa.rms_norm_fp8(dual(x, t(x)), w), lambda: nsa.quantize_rows_to_fp8(dual(x, t(x))),
        lambda: nsa.linear(dual(x, t(x)), sq), lambda: nsa.linear(x, dual(sq, t(sq))), lambda: nsa.linear(x, sq, dual(w, t(w))),
        lambda: nsa.linear(x, sq, residual=dual(x, t(x))), lambda: nsa.linear_fp8(e, k, es, ks, dual(w, t(w))), lambda: nsa.linear_fp8(e, k, dual(es, t(es)), ks),
        lambda: nsa.gated_mlp(dual(x, t(x)), sq, sq, sq), lambda: nsa.gated_mlp(x, sq, dual(v, t(v)), sq), lambda: nsa.gated_mlp(x, sq, sq, sq, residual=dual(x, t(x))),
        lambda: nsa.rope_axes_to_heads(dual(q, t(q)), q, q, pos, inv, (32,)), lambda: nsa.rope_axes_to_heads(q, q, dual(q, t(q)), pos, inv, (32,)),
    ]
    with fwad.dual_level():
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        nsa.linear(x, sq)                                                  # no tangent: as ever
