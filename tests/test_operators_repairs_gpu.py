"""gated_scan, dropout, sample_rows and their callers at calls that once went wrong: each against its 64-bit form or definition."""
import numpy as np
import pytest
import torch

import operator_forms as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from laed_amd import ops as _ops
    return _ops


def f64(t):
    return t.detach().double().cpu().numpy()


def sample_case(ops, rows, us, **kw):
    """rows [N,V] fp32 under one setting, every u of `us` for every row: the 64-bit form's tokens, and its log-probabilities to
    half a step of fp32 and the weights' fixed-point rounding (2^-44 of the largest weight each, V of them)."""
    N, V = rows.shape
    host = f64(rows)
    for u in us:
        ids, logp = ops.sample_rows(rows.cuda(), torch.full((N,), u, device="cuda"), return_logp=True, **kw)
        for r in range(N):
            tok, lp = F.sample_row(host[r], float(np.float32(u)), **kw)
            assert int(ids[r]) == tok, (r, u, kw, int(ids[r]), tok)
            assert abs(float(logp[r]) - lp) <= F.E * abs(lp) * 1.01 + V * 2.0 ** -44 + 1e-12, (r, u, kw, float(logp[r]), lp)


US = (0.0, 0.3, 0.77, 1.0 - 2.0 ** -24)


# ----------------------------------------------------------------------------------------------------------------
# a border of top-k or of the nucleus far below the largest logit and next to logit 0: the distance from the largest one is
# rounded by more than the logit itself
# ----------------------------------------------------------------------------------------------------------------
def border_rows(V, above, tops, tinies):
    """Rows with `above` logits from 0.05 to the largest one, the tiny ones next, all others from -1 down; shuffled alike."""
    rows = []
    for top in tops:
        for tiny in tinies:
            n = V - above - len(tiny)
            rows.append(torch.cat([torch.linspace(0.05, top, above), torch.tensor(tiny), torch.linspace(-1.0, -3.0, n)]))
    order = torch.randperm(V, generator=torch.Generator().manual_seed(V))
    return torch.stack(rows)[:, order]


TINY = ([1e-8], [-1e-8], [1e-8, 2e-8, -3e-8, 0.0, 1e-12], [4.7e-7, 3e-9, -4.7e-7, 1e-38], [1e-3, 1e-3 - 1e-9, 1e-3 - 1e-7])


@pytest.mark.parametrize("V", [2000, 5000, 30000])
def test_sample_top_k_border_next_to_zero(ops, V):
    rows = border_rows(V, 599, (8.0, 20.0, 11.328125), TINY)
    for k in (598, 599, 600, 601, 602, 604, 606):
        sample_case(ops, rows, US, top_k=k)
    sample_case(ops, rows, US[1:3], top_k=601, top_p=0.99, min_p=1e-6, temperature=1.7)


def test_sample_top_k_border_is_the_same_in_any_batch(ops):
    """255 rows of 2000 go to blocks of 1024 threads, 256 of them to blocks of 256: the same tokens, row by row."""
    rows = border_rows(2000, 599, (8.0,), TINY).repeat(52, 1)[:256].cuda()
    u = torch.rand(256, generator=torch.Generator().manual_seed(1)).cuda()
    for k in (300, 599, 600, 601, 603):
        one, logp1 = ops.sample_rows(rows, u, top_k=k, return_logp=True)
        two, logp2 = ops.sample_rows(rows[:255], u[:255], top_k=k, return_logp=True)
        assert torch.equal(one[:255], two) and torch.equal(logp1[:255], logp2) and (one >= 0).all()


def test_sample_top_k_border_of_normal_rows(ops):
    """N(0, 4) rows whose k-th logit lies near 0.1, the largest one near 8."""
    rows = torch.randn(48, 50000, generator=torch.Generator().manual_seed(11)) * 2
    for r in range(0, 48, 16):
        for k in sorted({int((rows[i] > 0.1).sum()) for i in range(r, r + 4)}):
            sample_case(ops, rows[r:r + 16], (0.4,), top_k=k)


@pytest.mark.parametrize("top,bin_", [(8.0, 300), (5.75, 700), (11.3, 1200)])
def test_sample_nucleus_border_next_to_zero(ops, top, bin_):
    """The temperature puts a bin's edge within fp64's rounding of logit 0; p crosses inside one of the tiny tokens' weights."""
    m = float(np.float32(top))
    tau = m / ((16 * bin_ - 0.5) * np.log(2.0) / 1024)
    tiny = np.concatenate([s * 10.0 ** np.arange(-18, -12, 0.25) for s in (1, -1)])
    row = np.concatenate([[m], np.linspace(m - 1, 1, 200), tiny, np.full(100, -5.0)]).astype(np.float32)
    rows = torch.from_numpy(row)[torch.randperm(len(row), generator=torch.Generator().manual_seed(bin_))][None]
    y = (np.sort(row.astype(np.float64))[::-1] - m) / tau
    mass = np.cumsum(np.exp(y))
    for j in range(200, 200 + len(tiny), 5):
        sample_case(ops, rows, (0.3, 1.0 - 2.0 ** -24), temperature=tau, top_p=float((mass[j] - np.exp(y[j]) / 2) / mass[-1]))


# ----------------------------------------------------------------------------------------------------------------
# more work than one grid of fewer than 2^32 threads holds
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("V,N", [(20, (1 << 24) + 5), (2100, (1 << 22) + 3)])
def test_sample_more_rows_than_a_grid_holds(ops, V, N):
    """One expanded row drawn from 2^24 times by 256 threads a row, 2^22 times by 1024: what calls of fewer rows draw."""
    row = torch.randn(1, V, generator=torch.Generator().manual_seed(V)).cuda()
    ids, logp = ops.sample_rows(row.expand(N, V), rng=(5, 9), temperature=0.7, top_p=0.9, return_logp=True)
    for lo in range(0, N, 1 << 20):
        hi = min(lo + (1 << 20), N)
        part, lpart = ops.sample_rows(row.expand(hi - lo, V), rng=(5, 9 + lo), temperature=0.7, top_p=0.9, return_logp=True)
        assert torch.equal(ids[lo:hi], part) and torch.equal(logp[lo:hi], lpart), lo
    assert ids.unique().numel() > 2


def spare_memory(gib):
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info()[0] > gib * 2.0 ** 30


def test_dropout_more_elements_than_a_grid_holds(ops):
    """2^34 + 5 elements that start off a vector boundary, single elements a thread: 32 GB of bf16, dropped in place."""
    from laed_amd._lib import check, lib, stream
    if not spare_memory(48):
        pytest.skip("needs 48 GB of device memory")
    n, p = (1 << 34) + 5, 0.25
    x = torch.ones(n + 2, device="cuda", dtype=torch.bfloat16)
    at = x[1:].data_ptr()
    assert at % 16
    check(lib.laed_dropout(at, 0, 0, None, 0, 0, at, 0, 0, 1, 1, n, 1, p, 7, 3, None, stream()), "laed_dropout")
    want = torch.tensor(1 / (1 - p), device="cuda").to(torch.bfloat16)
    for lo in (0, (1 << 33) - 4096, (1 << 34) - 5000, n - 9000):                # the first draws, both launches' ends, the last ones
        m = min(9000, n - lo)
        keep = ops.dropout_keep_mask(m, p, 7, 3 + lo, x.device) != 0
        assert torch.equal(x[1 + lo:1 + lo + m], torch.where(keep, want, torch.zeros_like(want))), lo
    assert float(x[0]) == 1 and float(x[n + 1]) == 1
    del x
    torch.cuda.empty_cache()


def test_dropout_lengths_around_a_block(ops):
    """Remainders of a vector, of a block's 1024 vectors and of both, forward over all of the tensor."""
    for n in (4095, 4096, 4097, 8191, 8192, 8193, 8195, 12288 + 1):
        for dt in (torch.float32, torch.bfloat16):
            x = torch.randn(n, device="cuda").to(dt)
            keep = ops.dropout_keep_mask(n, 0.5, 3, 4, x.device) != 0
            assert torch.equal(ops.dropout(x, 0.5, (3, 4)), torch.where(keep, x * 2, torch.zeros_like(x))), (n, dt)


@pytest.mark.parametrize("T,B,H,gib", [(1, 1 << 21, 2049, 100), (65, 209700, 2049, 190)])
def test_scan_more_channels_than_a_grid_holds(ops, T, B, H, gib):
    """One bf16 input expanded over the batch, one channel a thread: more than 2^31 threads, so two or three launches (T = 65: with
    two tiles on each one's tape).  Forward and backward; every sequence gives the numbers of a call of four."""
    if not spare_memory(gib):
        pytest.skip("needs %d GB of device memory" % gib)
    g = torch.Generator(device="cuda").manual_seed(3)
    gi = torch.randn(T, 1, 2 * H, device="cuda", generator=g).bfloat16()
    dout = torch.randn(T, 1, H, device="cuda", generator=g).bfloat16()
    few = gi.expand(T, 4, 2 * H).contiguous().requires_grad_(True)
    want, wantT = ops.gated_scan(few)
    dwant = torch.autograd.grad(want, few, dout.expand(T, 4, H))[0]
    x = gi.expand(T, B, 2 * H).requires_grad_(True)
    out, hT = ops.gated_scan(x)
    assert torch.equal(want[:, :1], want[:, 3:]) and torch.equal(dwant[:, :1], dwant[:, 3:])

    def same(a, b):
        step = max(1, (1 << 29) // (a.shape[0] * a.shape[2]))
        return all(bool((a[:, i:i + step] == b[:, :1]).all()) for i in range(0, B, step))

    assert same(out, want) and same(hT[None], wantT[None])
    del hT
    d = torch.autograd.grad(out, x, dout.expand(T, B, H))[0]
    assert same(d, dwant)
    del out, d, x
    torch.cuda.empty_cache()


# ----------------------------------------------------------------------------------------------------------------
# derivatives
# ----------------------------------------------------------------------------------------------------------------
def test_forward_mode_through_a_backward_pass_is_refused(ops):
    """A gradient that carries a tangent (forward over reverse) is refused as an input that carries one is."""
    import torch.autograd.forward_ad as forward_ad
    gi, x = torch.randn(4, 2, 6, device="cuda", requires_grad=True), torch.randn(30, device="cuda", requires_grad=True)
    with forward_ad.dual_level():
        for y, leaf in ((ops.gated_scan(gi)[0], gi), (ops.dropout(x, 0.5, (1, 2)), x)):
            d = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, d, retain_graph=True)
            assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].shape == leaf.shape
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.dropout(forward_ad.make_dual(x.detach(), torch.ones_like(x)), 0.5, (1, 2))


# ----------------------------------------------------------------------------------------------------------------
# temperatures as small as the logits
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [1e-20, 1e-30, 1e-41])
def test_sample_tiny_temperatures_of_tiny_logits(ops, scale):
    """What counts is the ratio: logits of 1e-30 under a temperature of 1e-30 (1e-41: subnormal ones) are far from equal."""
    rows = (torch.randn(4, 3000, generator=torch.Generator().manual_seed(5), dtype=torch.float64) * scale).float()
    for t in (0.3 * scale, scale, 5 * scale):
        for kw in ({}, {"top_p": 0.9}, {"top_k": 700, "min_p": 0.03}, {"top_k": 50, "top_p": 0.8}):
            sample_case(ops, rows, (0.2, 0.6, 0.95), temperature=t, **kw)
    ids = ops.sample_rows(rows.cuda(), torch.full((4,), 0.9, device="cuda"), temperature=5e-324)      # the smallest number there is
    assert torch.equal(ids.cpu(), rows.argmax(dim=1))


# ----------------------------------------------------------------------------------------------------------------
# dropout's factor
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("p", [0.6, 0.9, 0.99, 0.999, 1 - 1e-5])
def test_dropout_factor_of_large_p(ops, p):
    """1 / (1 - p) from p itself, not from p in fp32, forward and backward; the few that are kept decide by p in fp32."""
    n = 1 << 20
    x = torch.randn(n, device="cuda", requires_grad=True)
    y = ops.dropout(x, p, (21, 4))
    dy = torch.randn(n, device="cuda")
    dx = torch.autograd.grad(y, x, dy)[0]
    for got, src in ((y, x), (dx, dy)):
        want, err, keep = F.dropout(f64(src), p, 21, 4)
        assert keep.any() and (np.abs(f64(got) - want) <= err).all()


# ----------------------------------------------------------------------------------------------------------------
# modules
# ----------------------------------------------------------------------------------------------------------------
def test_two_modules_draw_different_masks():
    """Two dropouts, and the dropouts inside two stacks of the same weights: independent decisions (kept by both: p^2 of them)."""
    from laed_amd import nn_lib
    from laed_amd.enc2dec.base_modules import GatedRNN
    x, n = torch.ones(1 << 16, device="cuda"), 1 << 16
    a, b = nn_lib.Dropout(0.5), nn_lib.Dropout(0.5)
    both = float(((a(x) != 0) & (b(x) != 0)).double().mean())
    assert abs(both - 0.25) < 5 * (0.25 * 0.75 / n) ** 0.5         # 5 standard deviations
    stacks = [GatedRNN(6, 8, 2, dropout=0.5).cuda() for _ in range(2)]
    stacks[1].load_state_dict(stacks[0].state_dict())
    y = torch.randn(3, 9, 6, device="cuda")
    assert not torch.equal(stacks[0](y)[0], stacks[1](y)[0])
    assert torch.equal(stacks[0].eval()(y)[0], stacks[1].eval()(y)[0])


def test_unfiltered_sampling_of_the_gated_recurrence():
    """rnn_cell='glr' without filters: sample_rows over the whole vocabulary, one uniform number a row and step; other shapes of
    replayed numbers are refused."""
    from laed_amd import ops
    from laed_amd.enc2dec.decoders import GEN, DecoderRNN
    torch.manual_seed(1)
    V, E, H, B, L = 211, 8, 16, 5, 6
    dec = DecoderRNN(V, L, E, H, 2, 3, rnn_cell='glr').cuda().eval()
    with torch.no_grad():
        dec.project.weight.mul_(8.0)
    h0, u = torch.randn(1, B, H, device="cuda"), torch.rand(L, B)
    for replayed in (u, None):
        dec.injected_u, dec.sample_step = (None if replayed is None else u.numpy()), 3
        lazy, _, ret = dec(B, init_state=h0, mode=GEN, gen_type='sample')
        ids = torch.cat(ret[dec.KEY_SEQUENCE], dim=1).cpu().numpy()
        logits = f64(ops.sgemm(lazy.h_tm.reshape(L * B, H).contiguous(), dec.project.weight.detach(), transB=True, bias=dec.project.bias.detach()))
        for t in range(L):
            n = replayed[t] if replayed is not None else ops.uniform(B, dec.sample_seed * 1000003 + 3, t << 32, "cuda").cpu()
            assert ids[:, t].tolist() == [F.sample_row(logits[t * B + b], float(n[b]))[0] for b in range(B)], t
    for shape in ((L, B, V), (L + 1, B), (L, B + 1)):
        dec.injected_u = torch.rand(*shape).numpy()
        with pytest.raises(ValueError, match="max_len, B"):
            dec(B, init_state=h0, mode=GEN, gen_type='sample')


# ----------------------------------------------------------------------------------------------------------------
# nothing is written beside an output
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,B,H", [(1, 3, 5), (13, 2, 7), (65, 3, 33), (41, 2, 64), (1500, 2, 24), (1501, 1, 37)])
def test_scan_does_not_write_beside_its_outputs(T, B, H, dt):
    """The C entries on buffers with guards in front of, behind and (strided outputs) between the rows: out, dgi, hT, dh0, the tape
    and the scratch.  The numbers are the 64-bit form's, to its bounds."""
    from laed_amd._lib import check, lib, stream
    code, pad, guard = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt], 64, 7.0
    ws_n, tape_n = int(lib.laed_gated_scan_workspace(T, B, H)), int(lib.laed_gated_scan_tape(T, B, H))
    assert (ws_n > 0) == (T > 1000)
    g = torch.Generator(device="cuda").manual_seed(T)
    gi = torch.randn(T, B, 2 * H, device="cuda", generator=g).to(dt)
    h0 = torch.randn(B, H, device="cuda", generator=g)
    dout, dhT = torch.randn(T, B, H, device="cuda", generator=g).to(dt), torch.randn(B, H, device="cuda", generator=g)
    lengths = torch.tensor([T, T // 2, 0][:B], device="cuda")
    for lens, reverse in ((None, 0), (lengths, 1)):
        want = F.gated_scan(f64(gi), f64(h0), None if lens is None else lens.tolist(), bool(reverse), f64(dout), f64(dhT))
        for gap, off in ((0, 0), (8, 0), (3, 1)):
            def guarded(n, dtype=torch.float32):
                buf = torch.full((n + 2 * pad + off,), guard, device="cuda", dtype=dtype)
                return buf, buf[pad + off:pad + off + n]

            def rows(width):                                       # [T][B][width] with `gap` elements behind each row
                buf, mid = guarded(T * B * (width + gap), dt)
                return buf, mid.view(T, B, width + gap)

            (ob, o), (qb, q) = rows(H), rows(2 * H)
            (tb, tape), (wb, ws) = guarded(tape_n), guarded(ws_n)
            (hb, h), (db, d) = guarded(B * H), guarded(B * H)
            at = lambda t: None if t is None else t.data_ptr()     # noqa: E731
            scratch = (ws.data_ptr(), ws_n) if ws_n else (None, 0)
            check(lib.laed_gated_scan_fwd(at(gi), B * 2 * H, 2 * H, at(h0), at(lens), T, B, H, code, reverse, at(o), B * (H + gap), H + gap,
                                          at(h), at(tape), *scratch, stream()), "fwd")
            check(lib.laed_gated_scan_bwd(at(gi), B * 2 * H, 2 * H, at(tape), at(lens), at(dout), B * H, H, at(dhT), T, B, H, code, reverse,
                                          at(q), B * (2 * H + gap), 2 * H + gap, at(d), *scratch, stream()), "bwd")
            for got, name in ((o[..., :H], "out"), (q[..., :2 * H], "dgi"), (h.view(B, H), "hT"), (d.view(B, H), "dh0")):
                half = F.HALF_STEP[str(got.dtype).replace("torch.", "")]                 # one rounding to the output's type
                tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-38             # half of the smallest subnormal's place
                bound = want[name + "_err"] + half * (np.abs(want[name]) + want[name + "_err"]) * 1.001 + tiny
                assert (np.abs(f64(got) - want[name]) <= bound).all(), (name, gap, off)
            assert (o[..., H:] == guard).all() and (q[..., 2 * H:] == guard).all()
            for buf, n in ((ob, o.numel()), (qb, q.numel()), (tb, tape_n), (wb, ws_n), (hb, B * H), (db, B * H)):
                assert (buf[:pad + off] == guard).all() and (buf[pad + off + n:] == guard).all()
