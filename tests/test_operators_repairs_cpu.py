"""gated_scan, dropout, sample_rows and their callers without a GPU: calls that once lost a result in silence are refused, or do
what is documented."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture(scope="module")
def ops():
    from laed_amd import ops as _ops
    return _ops


def refused(match, fn, *a, **k):
    from laed_amd._lib import LaedError
    with pytest.raises(LaedError, match=match):
        fn(*a, **k)


def test_forward_mode_derivatives_are_refused(ops):
    """A tangent would be dropped, that is, taken for zero; with and without recording for reverse mode."""
    with forward_ad.dual_level():
        dual = lambda *s: forward_ad.make_dual(torch.ones(*s), torch.ones(*s))      # noqa: E731
        z = torch.zeros
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                refused("forward-mode", ops.gated_scan, dual(2, 3, 4))
                refused("forward-mode", ops.gated_scan, z(2, 3, 4), dual(3, 2))
                refused("forward-mode", ops.gated_scan_step, dual(3, 4), z(3, 2))
                refused("forward-mode", ops.gated_scan_step, z(3, 4), dual(3, 2))
                refused("forward-mode", ops.dropout, dual(4, 5), 0.5, (1, 0))
                refused("forward-mode", ops.dropout, z(4, 5), 0.5, (1, 0), residual=dual(4, 5))
                refused("forward-mode", ops.sample_rows, dual(3, 7), z(3), return_logp=True)
        refused("CPU tensor", ops.gated_scan, z(2, 3, 4))          # without a tangent: as before
        refused("CPU tensor", ops.dropout, z(4, 5), 0.5, (1, 0))
        refused("CPU tensor", ops.sample_rows, dual(3, 7), z(3))   # tokens have no derivative
    refused("CPU tensor", ops.gated_scan, z(2, 3, 4))


def test_results_without_a_graph_are_refused_while_one_is_recorded(ops):
    """The one-token forms and log-probabilities have no backward pass: inputs that require grad would be cut off in silence."""
    from laed_amd.enc2dec.base_modules import GatedRNN
    z = lambda *s: torch.zeros(*s, requires_grad=True)             # noqa: E731
    c = torch.zeros
    step = GatedRNN(5, 2).step
    refused("no backward pass", ops.gated_scan_step, z(3, 4), c(3, 2))
    refused("no backward pass", ops.gated_scan_step, c(3, 4), z(3, 2))
    refused("no backward pass", ops.gated_scan_step, c(3, 4), c(3, 2), h_out=z(3, 2))
    refused("no backward pass", step, z(3, 5), c(3, 2))
    refused("no backward pass", step, c(3, 5), z(3, 2))
    refused("no backward pass", ops.sample_rows, z(3, 7), c(3), return_logp=True)
    refused("CPU tensor", ops.sample_rows, z(3, 7), c(3))          # tokens alone
    with torch.no_grad():
        refused("CPU tensor", ops.gated_scan_step, z(3, 4), z(3, 2))
        refused("CPU tensor", ops.sample_rows, z(3, 7), c(3), return_logp=True)
