"""gated_scan, dropout and sample_rows on the GPU against their 64-bit forms (operator_forms.py)."""
import numpy as np
import pytest
import torch

import operator_forms as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def name(dt):
    return str(dt).replace("torch.", "")


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from laed_amd import ops as _ops
    return _ops


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, err, dt):
    """|got - want| within the fp32 bound and one rounding to the output's type (half a step of the value, and half of the
    smallest subnormal's place)."""
    half = F.HALF_STEP[name(dt)]
    tiny = 2.0 ** -25 if dt == torch.float16 else 1e-38
    bound = err + half * (np.abs(want) + err) * 1.001 + tiny
    bad = np.abs(f64(got) - want) - bound
    assert not (bad > 0).any() and np.isfinite(f64(got)).all(), (float(bad.max()), np.unravel_index(bad.argmax(), bad.shape))


# ----------------------------------------------------------------------------------------------------------------
# gated_scan
# ----------------------------------------------------------------------------------------------------------------
def scan_case(ops, T, B, H, dt, layout="time", lengths=None, h0=True, reverse=False, seed=0, bias=1.0, grad=True, dout=True, dhT=True):
    g = torch.Generator().manual_seed(seed)
    gi = torch.randn(T, B, 2 * H, generator=g)
    gi[..., :H] = gi[..., :H] * 1.5 + bias
    gi = gi.to(dt)
    if layout == "batch":
        dev = gi.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    elif layout == "sliced":                                       # a larger tensor's inside: odd strides, unaligned rows
        big = torch.full((T + 1, B + 2, 2 * H + 3), float("nan"), dtype=dt)
        big[:T, 1:B + 1, 1:2 * H + 1] = gi
        dev = big.cuda()[:T, 1:B + 1, 1:2 * H + 1]
    else:
        dev = gi.cuda()
    hs = torch.randn(B, H, generator=g) if h0 else None
    lens = None if lengths is None else torch.tensor(lengths)
    do = torch.randn(T, B, H, generator=g).to(dt) if dout else None
    dh = torch.randn(B, H, generator=g) if dhT else None
    n = lambda t: None if t is None else f64(t)                    # noqa: E731
    want = F.gated_scan(n(gi), n(hs), lengths, reverse, *([n(do), n(dh)] if grad else []))
    gin = dev.detach().requires_grad_(grad)
    hin = None if hs is None else hs.cuda().requires_grad_(grad)
    ldev = None if lens is None else lens.cuda()
    out, hT = ops.gated_scan(gin, hin, ldev, reverse)
    assert out.dtype == dt and hT.dtype == torch.float32 and tuple(out.shape) == (T, B, H)
    close(out, want["out"], want["out_err"], dt)
    close(hT, want["hT"], want["hT_err"], torch.float32)
    if lens is not None:
        pad = torch.arange(T)[:, None] >= lens[None]
        assert (out.cpu()[pad] == 0).all()
    if not grad:
        return
    outs = [(o, d.cuda()) for o, d in ((out, do), (hT, dh)) if d is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [t for t in (gin, hin) if t is not None], [d for _, d in outs])
    close(grads[0], want["dgi"], want["dgi_err"], dt)
    if hin is not None:
        close(grads[1], want["dh0"], want["dh0_err"], torch.float32)
    with torch.no_grad():                                          # without a tape: the same numbers
        out2, hT2 = ops.gated_scan(gin, hin, ldev, reverse)
    assert torch.equal(out2, out.detach()) and torch.equal(hT2, hT.detach())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,B,H", [(1, 1, 1), (1, 30, 512), (2, 3, 5), (7, 2, 130), (15, 4, 64), (16, 2, 256), (17, 3, 100), (40, 6, 512),
                                   (63, 1, 72), (64, 2, 8), (65, 5, 257), (129, 1, 1024), (300, 2, 96)])
def test_scan_sizes(ops, T, B, H, dt):
    scan_case(ops, T, B, H, dt, seed=T + H)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,B,H,layout", [(2500, 1, 40, "time"), (5000, 2, 64, "batch"), (1111, 3, 33, "batch"), (4097, 1, 128, "time")])
def test_scan_long(ops, T, B, H, layout, dt):
    scan_case(ops, T, B, H, dt, layout, seed=T)


def test_scan_remembers_over_thousands_of_steps(ops):
    """Gates that stay open (z = 0.9997): what a step adds is small beside the state, and errors live for thousands of steps."""
    scan_case(ops, 6000, 1, 64, torch.float32, bias=8.0, seed=1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["batch", "sliced"])
@pytest.mark.parametrize("T,B,H", [(9, 4, 24), (70, 3, 50), (33, 1, 16), (1, 4, 24)])
def test_scan_layouts(ops, T, B, H, layout, dt):
    scan_case(ops, T, B, H, dt, layout, seed=H)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_scan_lengths(ops, reverse, dt):
    scan_case(ops, 50, 6, 40, dt, lengths=[50, 0, 1, 16, 33, 49], reverse=reverse, seed=1)
    scan_case(ops, 50, 3, 40, dt, lengths=[70, -3, 20], reverse=reverse, seed=2)          # beyond either end
    scan_case(ops, 700, 3, 24, dt, "batch", lengths=[700, 64, 300], reverse=reverse, seed=3)
    scan_case(ops, 30, 2, 16, dt, lengths=[0, 0], reverse=reverse, seed=4)


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_optional_arguments(ops, reverse):
    for kw in ({"h0": False}, {"dout": False}, {"dhT": False}, {"h0": False, "dhT": False}):
        scan_case(ops, 41, 3, 20, torch.float32, reverse=reverse, seed=5, **kw)
        scan_case(ops, 400, 2, 12, torch.float32, reverse=reverse, seed=6, **kw)


def test_scan_empty(ops):
    h0 = torch.randn(3, 4, device="cuda", requires_grad=True)
    gi = torch.zeros(0, 3, 8, device="cuda", requires_grad=True)
    out, hT = ops.gated_scan(gi, h0)
    assert tuple(out.shape) == (0, 3, 4) and torch.equal(hT, h0)
    d = torch.randn(3, 4, device="cuda")
    dgi, dh0 = torch.autograd.grad(hT, (gi, h0), d)
    assert torch.equal(dh0, d) and dgi.numel() == 0
    assert tuple(ops.gated_scan(torch.zeros(4, 0, 8, device="cuda"))[0].shape) == (4, 0, 4)
    assert tuple(ops.gated_scan(torch.zeros(4, 3, 0, device="cuda"))[0].shape) == (4, 3, 0)


def test_scan_padding_is_never_read(ops):
    """NaN and infinities behind a sequence's end reach neither the outputs nor the gradients."""
    T, B, H = 90, 3, 32
    lengths = torch.tensor([90, 20, 0]).cuda()
    gi = torch.randn(T, B, 2 * H, device="cuda")
    pad = torch.arange(T, device="cuda")[:, None] >= lengths[None]
    dirty = gi.clone()
    dirty[pad] = float("nan")
    dirty[40:, 1, ::2] = float("inf")
    dout = torch.randn(T, B, H, device="cuda")
    ddirty = dout.clone()
    ddirty[pad] = float("nan")
    res = []
    for g, d in ((gi, dout), (dirty, ddirty)):
        g = g.clone().requires_grad_(True)
        out, hT = ops.gated_scan(g, None, lengths)
        res.append((out.detach(), hT.detach(), torch.autograd.grad(out, g, d)[0]))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_scan_saturated_gates(ops):
    """f = +-inf, +-200: the state is kept exactly, or replaced exactly."""
    gi = torch.zeros(4, 1, 8, device="cuda")
    gi[:, 0, :4] = torch.tensor([[float("inf")] * 4, [200.0] * 4, [-200.0] * 4, [float("-inf")] * 4], device="cuda")
    gi[:, 0, 4:] = torch.tensor([[5.0] * 4, [6.0] * 4, [7.0] * 4, [8.0] * 4], device="cuda")
    out, hT = ops.gated_scan(gi, torch.full((1, 4), 3.0, device="cuda"))
    assert out[:, 0, 0].tolist() == [3.0, 3.0, 7.0, 8.0] and hT[0, 0].item() == 8.0


def test_scan_broadcast_state_and_inputs(ops):
    """One initial state for all sequences, one gate for all sequences: gradients are summed over what was broadcast."""
    T, B, H = 20, 4, 16
    g1 = torch.randn(T, 1, 2 * H, device="cuda", requires_grad=True)
    h1 = torch.randn(1, H, device="cuda", requires_grad=True)
    dout = torch.randn(T, B, H, device="cuda")
    out, _ = ops.gated_scan(g1.expand(T, B, 2 * H), h1.expand(B, H))
    a = torch.autograd.grad(out, (g1, h1), dout)
    g2, h2 = g1.detach().expand(T, B, 2 * H).contiguous().requires_grad_(True), h1.detach().expand(B, H).contiguous().requires_grad_(True)
    b = torch.autograd.grad(ops.gated_scan(g2, h2)[0], (g2, h2), dout)
    # the same numbers, summed over B = 4 in fp32: 3 roundings of sums of magnitude <= sum |terms|
    assert ((a[0] - b[0].sum(1, keepdim=True)).abs() <= 4 * F.E * b[0].abs().sum(1, keepdim=True)).all()
    assert ((a[1] - b[1].sum(0, keepdim=True)).abs() <= 4 * F.E * b[1].abs().sum(0, keepdim=True)).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_scan_step_is_the_scan(ops, dt):
    """Token by token (new state each time, then in place) gives the sequence's fp32 states to their error bound."""
    T, B, H = 12, 30, 68
    gi = torch.randn(T, B, 2 * H, device="cuda").to(dt)
    h0 = torch.randn(B, H, device="cuda")
    want = F.gated_scan(f64(gi), f64(h0))
    h, hp = h0.clone(), h0.clone()
    for t in range(T):
        out, h = ops.gated_scan_step(gi[t], h)
        out2, same = ops.gated_scan_step(gi[t], hp, h_out=hp)
        assert same is hp and torch.equal(out, out2) and torch.equal(h, hp)
        close(out, want["out"][t], want["out_err"][t], dt)
    close(h, want["hT"], want["hT_err"], torch.float32)


def test_scan_step_refuses_overlapping_states(ops):
    from laed_amd._lib import LaedError
    buf = torch.zeros(5, 8, device="cuda")
    with pytest.raises(LaedError, match="overlaps"):
        ops.gated_scan_step(torch.zeros(4, 16, device="cuda"), buf[:4], h_out=buf[1:])
    with pytest.raises(LaedError, match="contiguous fp32"):
        ops.gated_scan_step(torch.zeros(4, 16, device="cuda"), buf[:4], h_out=torch.zeros(8, 4, device="cuda").t())


def test_scan_of_inputs_expanded_over_time(ops):
    g1 = torch.randn(1, 3, 16, device="cuda", requires_grad=True)
    out, hT = ops.gated_scan(g1.expand(30, 3, 16))
    g = torch.autograd.grad(out.sum(), g1)[0]
    g2 = g1.detach().repeat(30, 1, 1).requires_grad_(True)
    want, _ = ops.gated_scan(g2)
    assert torch.equal(out, want)
    d = torch.autograd.grad(want.sum(), g2)[0]
    assert ((g - d.sum(0, keepdim=True)).abs() <= 30 * F.E * d.abs().sum(0, keepdim=True)).all()


def test_scan_is_reproducible_and_leaves_neighbours_alone(ops):
    T, B, H = 500, 2, 40
    gi = torch.randn(T, B, 2 * H, device="cuda", requires_grad=True)
    dout = torch.randn(T, B, H, device="cuda")
    runs = []
    for _ in range(3):
        out, hT = ops.gated_scan(gi)
        runs.append((out.detach(), hT.detach(), torch.autograd.grad((out, hT), gi, (dout, torch.ones_like(hT)))[0]))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_scan_second_backward_and_no_double_backward(ops):
    gi = torch.randn(9, 2, 8, device="cuda", requires_grad=True)
    out, _ = ops.gated_scan(gi)
    a = torch.autograd.grad(out.sum(), gi, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(out.sum(), gi)[0])
    out, _ = ops.gated_scan(gi)
    d = torch.autograd.grad(out.sum(), gi, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        d.sum().backward()


# ----------------------------------------------------------------------------------------------------------------
# dropout
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (3, 7), (1200, 200), (65, 33), (2, 3, 4, 5), (4099,), (16, 8)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_sizes(ops, shape, dt, residual):
    p, seed, offset = 0.3, 123457, 1 << 33
    x = torch.randn(shape, device="cuda").to(dt).requires_grad_(True)
    r = torch.randn(shape, device="cuda").to(dt).requires_grad_(True) if residual else None
    y = ops.dropout(x, p, (seed, offset), residual=r)
    want, err, keep = F.dropout(f64(x), p, seed, offset, None if r is None else f64(r))
    close(y, want, err, dt)
    stored = ops.dropout_keep_mask(x.numel(), p, seed, offset, x.device).view(shape)
    assert np.array_equal(stored.cpu().numpy() != 0, keep)
    dy = torch.randn(shape, device="cuda").to(dt)
    grads = torch.autograd.grad(y, [x] if r is None else [x, r], dy)
    wdx, edx, _ = F.dropout(f64(dy), p, seed, offset)
    close(grads[0], wdx, edx, dt)
    assert (grads[0].cpu().numpy() if dt == torch.float32 else f64(grads[0]))[~keep].any() == False  # noqa: E712
    if r is not None:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("make", [lambda t: t.transpose(0, 1), lambda t: t[1:], lambda t: t[:, 1:, 1:], lambda t: t[:, ::2],
                                  lambda t: t[..., ::2], lambda t: t.permute(2, 0, 1), lambda t: t[:, :1].expand(6, 5, 9),
                                  lambda t: t[..., 1:]])
def test_dropout_strides_keep_the_logical_numbering(ops, make, dt):
    """A view draws what its contiguous copy draws; forward and backward, with and without a residual of other strides."""
    base = torch.randn(6, 5, 9, device="cuda").to(dt)
    x = make(base)
    res = torch.randn(x.shape, device="cuda").to(dt)
    for r in (None, res, make(torch.randn(6, 5, 9, device="cuda").to(dt))):
        a = ops.dropout(x, 0.4, (9, 7), residual=r)
        b = ops.dropout(x.contiguous(), 0.4, (9, 7), residual=None if r is None else r.contiguous())
        assert torch.equal(a, b)
    xv = x.detach().requires_grad_(True)
    dy = torch.randn(x.shape, device="cuda").to(dt)
    g = torch.autograd.grad(ops.dropout(xv, 0.4, (9, 7)), xv, dy)[0]
    assert torch.equal(g, ops.dropout(dy, 0.4, (9, 7)))


def test_dropout_edges(ops):
    x = torch.randn(1000, device="cuda")
    assert torch.equal(ops.dropout(x, 0.0, (1, 0)), x)
    assert (ops.dropout(x, 1.0, (1, 0)) == 0).all()
    assert ops.dropout(x[:0], 0.5, (1, 0)).numel() == 0
    bad = torch.full((4096,), float("nan"), device="cuda")
    bad[::2] = float("inf")
    keep = torch.from_numpy(F.keep_draws(3, 0, 4096) / 2.0 ** 24 >= 0.5).cuda()
    y = ops.dropout(bad, 0.5, (3, 0))
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    big = (1 << 64) - 3                                            # numbers wrap at 2^64
    want, err, _ = F.dropout(f64(x), 0.5, -5, big)
    close(ops.dropout(x, 0.5, (-5, big)), want, err, torch.float32)


def test_dropout_numbers_on_the_device(ops):
    x = torch.randn(3000, device="cuda", requires_grad=True)
    rng = torch.tensor([77, 5], device="cuda")
    y = ops.dropout(x, 0.3, rng)
    assert torch.equal(y, ops.dropout(x, 0.3, (77, 5)))
    dy = torch.randn_like(x)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], ops.dropout(dy, 0.3, (77, 5)))


def test_dropout_second_derivative_and_repeated_backward(ops):
    x = torch.randn(500, device="cuda", requires_grad=True)
    for rng in ((8, 1), torch.tensor([8, 1], device="cuda")):
        y = ops.dropout(x, 0.3, rng)
        dy = torch.randn(500, device="cuda", requires_grad=True)
        dx = torch.autograd.grad(y, x, dy, create_graph=True)[0]
        assert torch.equal(dx, ops.dropout(dy.detach(), 0.3, (8, 1)))
        v = torch.randn(500, device="cuda")
        assert torch.equal(torch.autograd.grad(dx, dy, v)[0], ops.dropout(v, 0.3, (8, 1)))
        assert torch.equal(torch.autograd.grad(y, x, v)[0], ops.dropout(v, 0.3, (8, 1)))


def test_dropout_shards_draw_the_whole_batchs_decisions(ops):
    x = torch.randn(8, 50, device="cuda")
    whole = ops.dropout(x, 0.3, (11, 400))
    parts = [ops.dropout(x[i:i + 2], 0.3, (11, 400 + i * 50)) for i in range(0, 8, 2)]
    assert torch.equal(whole, torch.cat(parts))


def test_dropout_does_not_write_beside_its_output(ops):
    from laed_amd._lib import check, lib, stream
    for n in (1, 5, 1023, 1025, 4099):
        for dt, code in ((torch.float32, 0), (torch.bfloat16, 1)):
            x = torch.randn(n + 16, device="cuda").to(dt)
            y = torch.full((n + 16,), 7.0, device="cuda", dtype=dt)
            for o in (0, 1, 8):
                y.fill_(7.0)
                check(lib.laed_dropout(x[o:].data_ptr(), 0, 0, None, 0, 0, y[o:].data_ptr(), 0, 0, 1, 1, n, code, 0.5, 1, 2, None, stream()), "d")
                assert (y[:o] == 7).all() and (y[o + n:] == 7).all()
                assert torch.equal(y[o:o + n], ops.dropout(x[o:o + n].clone(), 0.5, (1, 2)))


# ----------------------------------------------------------------------------------------------------------------
# sample_rows
# ----------------------------------------------------------------------------------------------------------------
def sample_case(ops, logits, u, dt=torch.float32, **kw):
    """Tokens equal the 64-bit form's; log-probabilities to half a step of fp32 and the weights' fixed-point rounding
    (2^-44 of the largest weight each, V of them; 64-bit sums beside it are smaller)."""
    logits = logits.to(dt)
    host, V = f64(logits), logits.shape[1]
    ids, logp = ops.sample_rows(logits, u, return_logp=True, **{k: (v.cuda() if torch.is_tensor(v) else v) for k, v in kw.items()})
    ids2 = ops.sample_rows(logits, u, **{k: (v.cuda() if torch.is_tensor(v) else v) for k, v in kw.items()})
    assert torch.equal(ids, ids2)
    for r in range(logits.shape[0]):
        one = {k: (float(v[r]) if torch.is_tensor(v) else v) for k, v in kw.items()}
        if "top_k" in one:
            one["top_k"] = int(one["top_k"])
        tok, lp = F.sample_row(host[r], float(u[r]), **one)
        assert int(ids[r]) == tok, (r, int(ids[r]), tok, one)
        if np.isfinite(lp):
            assert abs(float(logp[r]) - lp) <= F.E * abs(lp) * 1.01 + V * 2.0 ** -44 + 1e-12, (r, float(logp[r]), lp)
        else:
            assert float(logp[r]) == lp
    return ids


FILTERS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.05}, {"temperature": 1.3, "top_k": 50, "top_p": 0.8, "min_p": 0.01},
           {"top_k": 3, "top_p": 0.999}, {"top_p": 0.0}, {"temperature": 0.0}, {"min_p": 1.0}, {"top_k": 10 ** 9}]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 65, 257, 1000, 4096, 4097, 10004, 50000, 66001, 131075])
def test_sample_sizes(ops, V, dt):
    N = 5 if V > 4000 else 9
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = 2.0 * torch.randn(N, V, device="cuda", generator=g)
    u = torch.rand(N, device="cuda", generator=g)
    for kw in FILTERS:
        sample_case(ops, logits, u, dt, **kw)


def test_sample_settings_per_row(ops):
    N, V = 24, 3001
    g = torch.Generator().manual_seed(4)
    logits = 3.0 * torch.randn(N, V, generator=g)
    t = torch.rand(N, generator=g) * 1.5
    t[3], t[7] = 0.0, 1e-6
    k = torch.randint(0, 100, (N,), generator=g)
    k[5], k[6] = 0, 5000
    p, m = torch.rand(N, generator=g), torch.rand(N, generator=g) * 0.2
    p[2], p[4], m[8], m[9] = 1.0, 0.0, 0.0, 1.0
    u = torch.rand(N, generator=g).cuda()
    sample_case(ops, logits.cuda(), u, temperature=t, top_k=k, top_p=p, min_p=m)
    sample_case(ops, logits.cuda(), u, top_k=k)
    # values outside their ranges, as a device tensor may hold them: greedy, off, off, one token
    nan = float("nan")
    ids = ops.sample_rows(logits[:1].expand(6, V).cuda(), torch.full((6,), 0.999, device="cuda"),
                          temperature=torch.tensor([-1.0, nan, 1.0, 1.0, 1.0, 1.0]).cuda(), top_k=torch.tensor([0, 0, -4, 0, 0, 0]).cuda(),
                          top_p=torch.tensor([1.0, 1.0, 1.0, nan, -2.0, 5.0]).cuda(), min_p=torch.tensor([0.0, 0.0, 0.0, nan, 0.0, -1.0]).cuda())
    best, plain = int(logits[0].argmax()), F.sample_row(f64(logits[0]), float(np.float32(0.999)))[0]
    assert ids.tolist() == [best, best, plain, plain, best, plain]


def test_sample_masked_rows(ops):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    V = 700
    rows = torch.randn(8, V)
    rows[0] = -inf                                                 # nothing left
    rows[1] = nan
    rows[2] = -inf
    rows[2, 699] = -5.0                                            # one token
    rows[3, ::2] = nan                                             # NaN between real ones
    rows[4] = low                                                  # the type's lowest value everywhere: all equal
    rows[5, 100:] = low
    rows[6, 3], rows[6, 600] = inf, inf                            # infinities share everything
    rows[7] = -inf
    rows[7, 0], rows[7, 1] = low, low
    u = torch.rand(8).cuda()
    for kw in ({}, {"top_k": 5}, {"top_p": 0.5}, {"min_p": 0.1}, {"temperature": 0.3, "top_k": 300, "top_p": 0.7}, {"temperature": 0.0},
               {"temperature": 1e-30}, {"temperature": 1e30}):
        ids = sample_case(ops, rows.cuda(), u, **kw)
        assert ids[:3].tolist() == [-1, -1, 699]
        assert int(ids[6]) in (3, 600) and int(ids[3]) % 2 == 1
    half = torch.full((2, 300), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    half[1, 7] = -inf
    sample_case(ops, half.cuda(), u[:2], torch.bfloat16, top_k=7)


@pytest.mark.parametrize("V", [600, 5000, 30000])
def test_sample_ties(ops, V):
    """Equal logits: the lower index goes first, at a top-k border, at a nucleus border and in a block of thousands."""
    g = torch.Generator().manual_seed(V)
    flat = torch.zeros(V)
    two = torch.where(torch.rand(V, generator=g) < 0.5, 1.0, 0.5)
    few = torch.randint(-3, 4, (V,), generator=g).float()
    zeros = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)   # +0 and -0 are equal
    close_ = 1.0 + torch.randperm(V, generator=g).float() * 2.0 ** -23  # adjacent floats: one bin, more of them than are ranked at once
    close_[::3] = close_[1]
    logits = torch.stack([flat, two, few, zeros, close_]).cuda()
    for u in (0.0, 0.25, 0.5, 0.999999, float(torch.rand(1, generator=g))):
        uu = torch.full((5,), u, device="cuda")
        for kw in ({}, {"top_k": 3}, {"top_k": V // 2 + 1}, {"top_p": 0.5}, {"top_k": V - 1, "top_p": 0.25}, {"top_k": V // 3, "top_p": 0.9, "min_p": 0.5}):
            sample_case(ops, logits, uu, **kw)


def test_sample_top_k_borders(ops):
    """Sizes of top_k around the limits at which its tokens are finished by themselves, for both numbers of threads, alone and
    with the other filters, with distinct and with tied logits."""
    g = torch.Generator().manual_seed(6)
    for V in (700, 2000, 5000):
        logits = torch.randn(300 if V == 2000 else 4, V, generator=g).cuda()
        logits[1] = (logits[1] * 4).round() / 4
        u = torch.rand(logits.shape[0], generator=g).cuda()
        for k in (2, 63, 255, 256, 257, 400, 511, 512, 513, 600, V - 1):
            sample_case(ops, logits[:4] if V == 2000 and k != 257 else logits, u[:4] if V == 2000 and k != 257 else u, top_k=k)
            sample_case(ops, logits[:4], u[:4], top_k=k, top_p=0.9, min_p=0.02, temperature=0.8)


def test_sample_certain_tokens_have_log_probability_zero(ops):
    logits = torch.randn(6, 3000, device="cuda") * 3
    u = torch.rand(6, device="cuda")
    for kw in ({"top_k": 1}, {"top_p": 0.0}, {"min_p": 1.0}, {"temperature": 0.0}, {"temperature": 1e-30}, {"top_k": 1, "top_p": 0.5, "temperature": 0.344}):
        ids, logp = ops.sample_rows(logits, u, return_logp=True, **kw)
        assert torch.equal(ids, logits.argmax(dim=1)) and (logp == 0).all(), kw


def test_sample_spread_logits(ops):
    """Logits spread over hundreds of units and masked by large negative numbers: borders far below the largest one."""
    g = torch.Generator().manual_seed(9)
    rows = torch.randn(4, 6000, generator=g) * torch.tensor([10.0, 40.0, 3.0, 3.0])[:, None]
    rows[2, 1000:] = -1e4
    rows[3, ::2] = -1e4
    u = torch.rand(4, generator=g).cuda()
    for kw in ({"top_k": 50}, {"top_k": 4000}, {"top_k": 2500, "top_p": 0.99}, {"top_p": 0.999}, {"temperature": 20.0, "top_k": 1500, "top_p": 0.9},
               {"temperature": 50.0, "top_p": 0.7}):
        sample_case(ops, rows.cuda(), u, **kw)
        sample_case(ops, rows.cuda(), u, torch.bfloat16, **kw)


def test_sample_wide_and_narrow_ranges(ops):
    g = torch.Generator().manual_seed(8)
    V = 20000
    rows = torch.stack([torch.randn(V, generator=g) * 1e30, torch.randn(V, generator=g) * 1e-30, torch.randn(V, generator=g) * 300,
                        torch.linspace(-80, 80, V), torch.randn(V, generator=g) + 3e4]).cuda()
    u = torch.rand(5, generator=g).cuda()
    for kw in ({}, {"top_k": 15000}, {"top_k": 2}, {"top_p": 0.99}, {"temperature": 100.0, "top_p": 0.6}, {"temperature": 0.01, "top_k": 12000, "top_p": 0.95}):
        sample_case(ops, rows, u, **kw)


def test_sample_uniform_numbers(ops):
    """u outside [0, 1) and NaN are clamped; the generator's draws are those of ops.uniform."""
    V = 333
    row = torch.randn(1, V)
    row[0, 0], row[0, V - 1] = -float("inf"), -float("inf")
    us = torch.tensor([0.0, -1.0, float("nan"), 1.0, 7.0, float("inf"), 1.0 - 2.0 ** -24, 1e-30])
    ids = sample_case(ops, row.expand(8, V).contiguous().cuda(), us.cuda())
    assert ids[:3].tolist() == [1, 1, 1] and ids[3:7].tolist() == [V - 2] * 4
    logits = torch.randn(50, V, device="cuda")
    a = ops.sample_rows(logits, rng=(99, 12), top_p=0.9)
    b = ops.sample_rows(logits, ops.uniform(50, 99, 12, "cuda"), top_p=0.9)
    c = torch.cat([ops.sample_rows(logits[i:i + 10], rng=(99, 12 + i), top_p=0.9) for i in range(0, 50, 10)])
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dt", DTYPES)
def test_sample_strides(ops, dt):
    """Rows inside a wider buffer, unaligned starts, expanded and transposed logits; what lies beside a row is never drawn."""
    for V, ld, off in ((1000, 1016, 0), (1000, 1003, 1), (37, 41, 3), (5001, 5008, 7)):
        buf = torch.full((6, ld), 1e4).to(dt).cuda()
        inner = torch.randn(6, V).to(dt)
        buf[:, off:off + V] = inner.cuda()
        u = torch.rand(6).cuda()
        view = buf[:, off:off + V]
        for kw in ({}, {"top_k": 20, "top_p": 0.9}):
            want = [F.sample_row(f64(inner[r]), float(u[r]), **kw)[0] for r in range(6)]
            assert ops.sample_rows(view, u, **kw).tolist() == want
            assert ops.sample_rows(view.t().contiguous().t(), u, **kw).tolist() == want
    one = torch.randn(1, 300).to(dt).cuda()
    u = torch.rand(4).cuda()
    assert torch.equal(ops.sample_rows(one.expand(4, 300), u), ops.sample_rows(one.expand(4, 300).contiguous(), u))


def test_sample_empty(ops):
    ids, logp = ops.sample_rows(torch.zeros(0, 5, device="cuda"), torch.zeros(0, device="cuda"), return_logp=True)
    assert ids.numel() == 0 and logp.numel() == 0 and ids.dtype == torch.int64


def test_sample_follows_the_distribution(ops):
    """10^5 draws of one row: each token's count within 6 standard deviations of its filtered probability."""
    n, V = 100000, 20
    row = torch.randn(V)
    p = torch.softmax(row.double() / 0.8, 0)
    top = torch.topk(p, 7)
    want = torch.zeros(V, dtype=torch.float64).scatter(0, top.indices, top.values / top.values.sum()).numpy()
    ids = ops.sample_rows(row.cuda().expand(n, V), rng=(31, 0), temperature=0.8, top_k=7)
    got = np.bincount(ids.cpu().numpy(), minlength=V)
    assert (np.abs(got - n * want) <= 6 * np.sqrt(n * want * (1 - want)) + 1e-9).all()


# ----------------------------------------------------------------------------------------------------------------
# streams, captured graphs, and the three together
# ----------------------------------------------------------------------------------------------------------------
def generator_step(ops, W, emb, proj, ids, h, u, rng):
    """One token of a recurrent generator: embedding, dropout (as in sampling with noise), gate product, step, logits, token."""
    x = ops.dropout(emb[ids], 0.1, rng)
    out, _ = ops.gated_scan_step(ops.sgemm(x, W, transB=True), h, h_out=h)
    return ops.sample_rows(ops.sgemm(out, proj, transB=True), u, temperature=0.8, top_k=30, top_p=0.95, min_p=0.01)


def test_the_three_together_match_the_forms(ops):
    """A training pass of a two-layer stack and a generation loop, each stage held to its 64-bit form on the stage's own input."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T, B, E, H, V = 23, 6, 24, 32, 501
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)     # noqa: E731
    x, W1, W2, lengths = r(T, B, E), r(2 * H, E) / 5, r(2 * H, H) / 6, torch.tensor([23, 1, 0, 12, 16, 22], device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, W1, W2)]
    gi1 = ops.linear(x.view(T * B, E), W1).view(T, B, 2 * H)
    o1, _ = ops.gated_scan(gi1, None, lengths)
    d1 = ops.dropout(o1, 0.25, (5, 0))
    gi2 = ops.linear(d1.view(T * B, H), W2).view(T, B, 2 * H)
    o2, h2 = ops.gated_scan(gi2, None, lengths)
    y = ops.dropout(o2, 0.25, (6, 0), residual=d1)
    f1, f2 = F.gated_scan(f64(gi1), None, lengths.tolist()), F.gated_scan(f64(gi2), None, lengths.tolist())
    close(o1, f1["out"], f1["out_err"], torch.float32)
    close(d1, *F.dropout(f64(o1), 0.25, 5, 0)[:2], torch.float32)
    close(o2, f2["out"], f2["out_err"], torch.float32)
    close(y, *F.dropout(f64(o2), 0.25, 6, 0, f64(d1))[:2], torch.float32)
    dy, dh = r(T, B, H), r(B, H)
    grads = torch.autograd.grad((y, h2), leaves, (dy, dh))
    # the chain in 64 bits from the formulas: products, dropout and recurrence backwards (tolerance: products of H or T*B
    # terms in fp32, 2^-24 sqrt(n) each in the mean, through two layers: 1e-5 of the largest entry leaves a factor of ten)
    k1, k2 = F.keep_draws(5, 0, T * B * H).reshape(T, B, H) / 2.0 ** 24 >= 0.25, F.keep_draws(6, 0, T * B * H).reshape(T, B, H) / 2.0 ** 24 >= 0.25
    do2 = np.where(k2, f64(dy) / 0.75, 0)
    dgi2 = F.gated_scan(f64(gi2), None, lengths.tolist(), False, do2, f64(dh))["dgi"].reshape(T * B, 2 * H)
    dd1 = (dgi2 @ f64(W2)).reshape(T, B, H) + f64(dy)
    dgi1 = F.gated_scan(f64(gi1), None, lengths.tolist(), False, np.where(k1, dd1 / 0.75, 0), None)["dgi"].reshape(T * B, 2 * H)
    wants = ((dgi1 @ f64(W1)).reshape(T, B, E), dgi1.T @ f64(x).reshape(T * B, E), dgi2.T @ f64(d1).reshape(T * B, H))
    for got, want in zip(grads, wants):
        assert np.abs(f64(got) - want).max() <= 1e-5 * np.abs(want).max()
    emb, proj = r(V, E), r(V, H)
    ids, h = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, H, device="cuda")
    for t in range(8):
        u = torch.rand(B, device="cuda", generator=g)
        before = h.clone()
        new = generator_step(ops, W1.detach(), emb, proj, ids, h, u, (7, t * B * E))
        xs = ops.dropout(emb[ids], 0.1, (7, t * B * E))
        want = F.gated_scan(f64(ops.sgemm(xs, W1.detach(), transB=True))[None], f64(before))
        close(h, want["hT"], want["hT_err"], torch.float32)
        logits = f64(ops.sgemm(h, proj, transB=True))
        assert new.tolist() == [F.sample_row(logits[b], float(u[b]), 0.8, 30, 0.95, 0.01)[0] for b in range(B)]
        ids = new


def test_on_another_stream(ops):
    """Launched on a side stream behind slow work: the operators run in that stream's order."""
    side = torch.cuda.Stream()
    gi, logits, u = torch.randn(300, 2, 64, device="cuda"), torch.randn(7, 9000, device="cuda"), torch.rand(7, device="cuda")
    want = (ops.gated_scan(gi)[0], ops.dropout(gi, 0.5, (1, 2)), ops.sample_rows(logits, u, top_p=0.9))
    big = torch.randn(4096, 4096, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, l = torch.zeros_like(gi), torch.zeros_like(logits)
        for _ in range(8):
            big = big @ big * 1e-3
        a.copy_(gi)
        l.copy_(logits)
        got = (ops.gated_scan(a)[0], ops.dropout(a, 0.5, (1, 2)), ops.sample_rows(l, u, top_p=0.9))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def captured(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_generation(ops):
    """Two captured steps of different sizes, replayed in turn with eager work between them: every replay equals the eager run."""
    g = torch.Generator(device="cuda").manual_seed(2)
    cases = []
    for B, V in ((5, 3000), (3, 70001)):
        E, H = 16, 40
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        W, emb, proj = r(2 * H, E) / 4, r(V, E), r(V, H)
        st = {"ids": torch.zeros(B, dtype=torch.int64, device="cuda"), "h": torch.zeros(B, H, device="cuda"), "u": torch.zeros(B, device="cuda"),
              "rng": torch.tensor([7, 0], device="cuda")}

        def step(W=W, emb=emb, proj=proj, st=st):
            st["ids"].copy_(generator_step(ops, W, emb, proj, st["ids"], st["h"], st["u"], st["rng"]))
            return st["ids"]

        graph, _ = captured(step)
        cases.append((graph, step, st, B))
    for graph, step, st, B in cases:
        st["ids"].zero_(), st["h"].zero_(), st["rng"][1].zero_()
    history = [[] for _ in cases]
    for t in range(6):
        for i, (graph, step, st, B) in enumerate(cases):
            st["u"].copy_(torch.rand(B, device="cuda", generator=g))
            st["rng"][1] = 1000 * t
            before = {k: v.clone() for k, v in st.items()}
            graph.replay()
            got = (st["ids"].clone(), st["h"].clone())
            torch.cuda.synchronize()
            for k, v in before.items():
                st[k].copy_(v)
            step()
            assert torch.equal(got[0], st["ids"]) and torch.equal(got[1], st["h"]), (i, t)
            history[i].append(got[0])
    assert any(not torch.equal(a, b) for a, b in zip(history[0], history[0][1:]))


def test_captured_training(ops):
    """Forward and backward of the recurrence and of dropout inside graphs (short and long time axes), replayed with new inputs and
    new random numbers; the leaves have no eager graph alive."""
    for T, B, H in ((40, 6, 32), (3000, 1, 64)):
        src, dout = torch.randn(T, B, 2 * H, device="cuda"), torch.randn(T, B, H, device="cuda")
        rng = torch.tensor([3, 0], device="cuda")
        gi = src.clone().requires_grad_(True)

        def step():
            out, hT = ops.gated_scan(gi)
            y = ops.dropout(out, 0.2, rng)
            return (y.detach(), hT.detach()) + torch.autograd.grad((y, hT), gi, (dout, torch.ones_like(hT)))

        graph, got = captured(step)
        for i in range(4):
            with torch.no_grad():
                gi.copy_(torch.randn(T, B, 2 * H, device="cuda"))
                rng[1] = 100 * i
            graph.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in got]
            torch.randn(1 << 20, device="cuda").sum().item()
            with torch.no_grad():
                fresh = gi.detach().clone()
            fresh.requires_grad_(True)
            out, hT = ops.gated_scan(fresh)
            y = ops.dropout(out, 0.2, (3, 100 * i))
            want = (y, hT) + torch.autograd.grad((y, hT), fresh, (dout, torch.ones_like(hT)))
            for a, b in zip(kept, want):
                assert torch.equal(a, b)
            del out, hT, y, want
