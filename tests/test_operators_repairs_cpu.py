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


def test_modules_without_a_seed_draw_from_streams_of_their_own(ops, monkeypatch):
    """(seed, offset) that each module hands to the operator: distinct between modules, layers and steps; unchanged for the first
    stack of a program; given seeds are kept."""
    import copy
    import weakref
    from laed_amd import nn_lib
    from laed_amd.enc2dec.base_modules import GatedRNN
    monkeypatch.setattr(nn_lib.DropoutStream, "held", weakref.WeakValueDictionary())
    seen = []
    monkeypatch.setattr(ops, "dropout", lambda x, p, rng, residual=None: seen.append(rng[0] & (2 ** 64 - 1)) or x)

    def draws(m):
        del seen[:]
        for d in (m.drop if isinstance(m, GatedRNN) else [m]):
            d(torch.zeros(2, 3))
        return list(seen)

    first, second = GatedRNN(4, 4, 4, dropout=0.5), GatedRNN(4, 4, 4, dropout=0.5)
    a, b, twin = nn_lib.Dropout(), nn_lib.Dropout(), copy.deepcopy(second)
    repr(first)                                                    # looking at a module takes no number
    first.eval()
    assert draws(first) == []
    first.train()
    assert draws(first) == [(2468 + i) * 1000003 for i in range(3)]
    got = [draws(m) for m in (first, second, a, b, twin, second, a)]
    assert got[0] == [(2468 + i) * 1000003 + 1 for i in range(3)]
    flat = sum(got, [])
    assert len(set(flat)) == len(flat)
    later = copy.deepcopy(second)                                  # has drawn twice: goes on as the original does
    assert draws(later) == draws(second)
    held = second.drop[0].seed
    del second
    assert later.drop[0].seed == held and nn_lib.Dropout().seed not in (held, a.seed, b.seed)
    assert draws(nn_lib.Dropout(0.5, seed=5)) == draws(nn_lib.Dropout(0.5, seed=5)) == [5 * 1000003]
    a.seed = 7
    a.step = 3
    assert draws(a) == [7 * 1000003 + 3]
    del first, later, b, twin                                      # built anew, the old ones gone: the same masks
    anew = GatedRNN(4, 4, 4, dropout=0.5)
    assert draws(anew) == [(2468 + i) * 1000003 for i in range(3)]


@pytest.mark.parametrize("cell", ["gru", "glr"])
@pytest.mark.parametrize("kw", [{"temperature": 0.5}, {"top_k": 3}, {"top_p": 0.9}, {"min_p": 0.1}])
def test_filters_are_refused_where_nothing_is_drawn(cell, kw):
    """Beam search, greedy decoding and teacher forcing would ignore them."""
    from laed_amd.enc2dec.decoders import GEN, TEACH_FORCE, DecoderRNN
    dec = DecoderRNN(11, 4, 5, 6, 2, 3, rnn_cell=cell)
    for mode, gen_type in ((GEN, 'beam'), (GEN, 'greedy'), (TEACH_FORCE, 'greedy'), (TEACH_FORCE, 'beam')):
        with pytest.raises(ValueError, match="belong to gen_type='sample'"):
            dec(2, inputs=torch.zeros(2, 3, dtype=torch.int64), init_state=torch.zeros(1, 2, 6), mode=mode, gen_type=gen_type, **kw)


def test_sizes_beyond_32_bits_are_refused(ops):
    """Expanded tensors reach them in little memory; the C entries would see the low 32 bits."""
    n, z = 2 ** 32 + 5, torch.zeros
    refused("must be below 2.31", ops.gated_scan, z(1, 1, 2).expand(1, n, 2))
    refused("must be below 2.31", ops.gated_scan, z(1, 1, 2).expand(n, 1, 2))
    refused("must be below 2.31", ops.gated_scan, z(1, 1, 1).expand(1, 1, 2 * n))
    refused("must be below 2.31", ops.gated_scan_step, z(1, 2).expand(n, 2), z(1, 1).expand(n, 1))
    refused("must be below 2.31", ops.sample_rows, z(1, 1).expand(1, n), z(1))


def test_channels_that_no_grid_holds_are_refused():
    """One sequence's threads, H times the waves of a block, have to fit a grid (H <= 2^28 always does)."""
    from laed_amd._lib import lib
    one = 16 << 20
    assert lib.laed_gated_scan_fwd(one, 0, 0, None, None, 57, 1, 2 ** 29, 1, 0, one, 0, 0, None, None, None, 0, None) == -1
    assert b"H too large" in lib.laed_last_error()
    assert lib.laed_gated_scan_bwd(one, 0, 0, one, None, None, 0, 0, None, 9, 1, 2 ** 31 - 1, 1, 0, one, 0, 0, None, None, 0, None) == -1
    assert b"H too large" in lib.laed_last_error()


def test_filters_of_a_greedy_decode_loop_are_refused(ops):
    w = [torch.zeros(*s) for s in ((11, 5), (18, 5), (18, 6), (18,), (18,), (11, 6), (11,), (2, 6))]
    with pytest.raises(ValueError, match="belong to sample=True"):
        ops.decode_greedy(*w, 4, 2, filters={"top_k": 3})
