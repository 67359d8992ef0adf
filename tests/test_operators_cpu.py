"""gated_scan, dropout and sample_rows without a GPU: refused arguments (Python and C entries), and the 64-bit forms the GPU
tests compare with -- their gradients against differences, their sampler against counts."""
import numpy as np
import pytest
import torch

import operator_forms as F


@pytest.fixture(scope="module")
def ops():
    from laed_amd import ops as _ops
    return _ops


def refused(match, fn, *a, **k):
    from laed_amd._lib import LaedError
    with pytest.raises(LaedError, match=match):
        fn(*a, **k)


def test_gated_scan_refusals(ops):
    z = torch.zeros
    refused("must be .T,B,2H", ops.gated_scan, z(3, 4))
    refused("must be .T,B,2H", ops.gated_scan, z(2, 3, 5))
    refused("expected float32", ops.gated_scan, z(2, 3, 4, dtype=torch.float64))
    refused("h0 must be", ops.gated_scan, z(2, 3, 4), z(3, 3))
    refused("lengths must be", ops.gated_scan, z(2, 3, 4), None, z(2, dtype=torch.int64))
    refused("lengths must be", ops.gated_scan, z(2, 3, 4), None, z(3))
    refused("CPU tensor", ops.gated_scan, z(2, 3, 4))
    refused("must be .B,2H", ops.gated_scan_step, z(2, 3, 4), z(3, 2))
    refused("must be .B,2H", ops.gated_scan_step, z(3, 5), z(3, 2))
    refused("h must be a contiguous fp32 .B,H. state", ops.gated_scan_step, z(3, 4), z(3, 4))
    refused("h must be a contiguous fp32 .B,H. state", ops.gated_scan_step, z(3, 4), z(3, 2, dtype=torch.bfloat16))
    refused("h_out must be", ops.gated_scan_step, z(3, 4), z(3, 2), z(2, 3).t())
    refused("CPU tensor", ops.gated_scan_step, z(3, 4), z(3, 2))


def test_dropout_refusals(ops):
    x = torch.zeros(4, 5)
    refused("p must lie", ops.dropout, x, -0.1, (1, 0))
    refused("p must lie", ops.dropout, x, 1.5, (1, 0))
    refused("p must lie", ops.dropout, x, float("nan"), (1, 0))
    refused("expected float32", ops.dropout, x.long(), 0.5, (1, 0))
    refused("residual must have", ops.dropout, x, 0.5, (1, 0), residual=torch.zeros(5, 4))
    refused("residual must have", ops.dropout, x, 0.5, (1, 0), residual=x.bfloat16())
    refused("rng", ops.dropout, x, 0.5, 7)
    refused("rng tensor", ops.dropout, x, 0.5, torch.zeros(2))
    refused("CPU tensor", ops.dropout, x, 0.5, (1, 0))


def test_sample_rows_refusals(ops):
    l, u = torch.zeros(3, 7), torch.zeros(3)
    refused("must be .N,V", ops.sample_rows, l[0], u)
    refused("must be .N,V", ops.sample_rows, l[:, :0], u)
    refused("expected float32", ops.sample_rows, l.double(), u)
    refused("either u or rng", ops.sample_rows, l)
    refused("either u or rng", ops.sample_rows, l, u, (1, 0))
    refused("u must be", ops.sample_rows, l, u[:2])
    refused("u must be", ops.sample_rows, l, u.double())
    refused("temperature must lie", ops.sample_rows, l, u, temperature=-1.0)
    refused("temperature must lie", ops.sample_rows, l, u, temperature=float("nan"))
    refused("top_k must lie", ops.sample_rows, l, u, top_k=-1)
    refused("whole number", ops.sample_rows, l, u, top_k=2.5)
    refused("top_p must lie", ops.sample_rows, l, u, top_p=1.5)
    refused("min_p must lie", ops.sample_rows, l, u, min_p=-0.5)
    refused("top_p per row", ops.sample_rows, l, u, top_p=torch.ones(4))
    refused("CPU tensor", ops.sample_rows, l, u)


def test_c_entries_check_their_arguments():
    from laed_amd._lib import lib
    assert lib.laed_gated_scan_tape(0, 4, 4) == 0 and lib.laed_gated_scan_tape(1, 4, 5) >= 20
    assert lib.laed_gated_scan_fwd(None, 0, 0, None, None, -1, 1, 1, 0, 0, None, 0, 0, None, None, None, 0, None) == -1
    assert lib.laed_gated_scan_fwd(None, 0, 0, None, None, 1, 1, 1, 3, 0, None, 0, 0, None, None, None, 0, None) == -1
    assert lib.laed_gated_scan_fwd(None, 0, 0, None, None, 1, 1, 1, 0, 0, None, 0, 0, None, None, None, 0, None) == -1
    assert b"null" in lib.laed_last_error()
    assert lib.laed_gated_scan_fwd(None, 0, 0, None, None, 5, 0, 4, 0, 0, None, 0, 0, None, None, None, 0, None) == 0
    assert lib.laed_gated_scan_bwd(None, 0, 0, None, None, None, 0, 0, None, 1, 1, 1, 0, 0, None, 0, 0, None, None, 0, None) == -1
    one = 16 * (1 << 20)                                           # few channels and a long time axis need scratch
    assert lib.laed_gated_scan_workspace(40, 60, 512) == 0 and lib.laed_gated_scan_workspace(1 << 20, 1, 8) > 0
    assert lib.laed_gated_scan_fwd(one, 16, 16, None, None, 1 << 20, 1, 8, 0, 0, one, 8, 8, None, None, None, 0, None) == -1
    assert b"workspace" in lib.laed_last_error()
    d = lib.laed_dropout
    assert d(None, 0, 0, None, 0, 0, None, 0, 0, 1, 1, 4, 0, 0.5, 0, 0, None, None) == -1
    assert d(None, 0, 0, None, 0, 0, None, 0, 0, 1, 1, 4, 0, 1.5, 0, 0, None, None) == -1
    assert d(None, 0, 0, None, 0, 0, None, 0, 0, 1, 1, -4, 0, 0.5, 0, 0, None, None) == -1
    assert d(None, 0, 0, None, 0, 0, None, 0, 0, 1, 1, 4, 9, 0.5, 0, 0, None, None) == -1
    assert d(None, 0, 0, None, 0, 0, None, 0, 0, 1, 0, 4, 0, 0.5, 0, 0, None, None) == 0
    s = lib.laed_sample_rows
    assert s(None, 4, 2, 4, 0, None, 0, 0, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None, None) == -1
    assert s(None, 4, 2, 0, 0, None, 0, 0, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None, None) == -1
    assert s(None, 4, 2, 4, 0, None, 0, 0, -1.0, None, 0, None, 1.0, None, 0.0, None, None, None, None) == -1
    assert s(None, 4, 2, 4, 0, None, 0, 0, 1.0, None, 0, None, 2.0, None, 0.0, None, None, None, None) == -1
    assert s(None, 4, 0, 4, 0, None, 0, 0, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None, None) == 0


def test_library_holds_no_packed_fp32_arithmetic(tmp_path):
    """Packed fp32 instructions are switched off in the build: none in the built device code."""
    import os
    import shutil
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "tools"))
    import check_mfma_hazards as H
    if not os.path.exists(os.path.join(H.LLVM, "llvm-objdump")):
        pytest.skip("no llvm-objdump in this image")
    local = shutil.copy(os.path.join(H.PKG, "liblaed_hip.so"), str(tmp_path / "lib.so"))
    subprocess.run([os.path.join(H.LLVM, "llvm-objdump"), "--offloading", local], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    parts = [p for p in os.listdir(str(tmp_path)) if p.endswith("gfx950")]
    assert parts
    for part in parts:
        txt = subprocess.run([os.path.join(H.LLVM, "llvm-objdump"), "-d", str(tmp_path / part)], check=True, stdout=subprocess.PIPE,
                             universal_newlines=True).stdout
        assert "v_fma_f32" in txt or "v_fmac_f32" in txt or "s_endpgm" in txt
        assert not any(op in txt for op in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_form_gradients_against_differences(reverse):
    rs = np.random.RandomState(3)
    T, B, H = 5, 3, 2
    gi, h0, dout, dhT = rs.randn(T, B, 2 * H), rs.randn(B, H), rs.randn(T, B, H), rs.randn(B, H)
    lengths = [5, 0, 3]

    def value(gi, h0):
        r = F.gated_scan(gi, h0, lengths, reverse)
        return (r["out"] * dout).sum() + (r["hT"] * dhT).sum()

    r = F.gated_scan(gi, h0, lengths, reverse, dout, dhT)
    for at, grad in ((gi, r["dgi"]), (h0, r["dh0"])):
        num = np.zeros_like(at)
        for i in np.ndindex(at.shape):
            keep, step = at[i], 1e-6
            at[i] = keep + step
            hi = value(gi, h0)
            at[i] = keep - step
            lo = value(gi, h0)
            at[i] = keep
            num[i] = (hi - lo) / (2 * step)
        # central differences: truncation ~ step^2, cancellation ~ 2^-52 |value| / step
        assert np.abs(num - grad).max() < 1e-8


def test_draws_are_the_generators():
    """Known values of the hash, and the share of draws below a border (n = 2^16: 5 standard deviations are 0.0098)."""
    a, b = F.keep_draws(5, 1000, 8), F.keep_draws(5, 1004, 4)
    assert (a[4:] == b).all() and a.min() >= 0 and a.max() < 2 ** 24
    assert abs(float((F.keep_draws(77, 0, 1 << 16) < 0.3 * 2 ** 24).mean()) - 0.3) < 0.0098 * 0.92


def test_sampler_form_counts():
    """Tokens drawn for evenly spread u appear in proportion to the filtered probabilities (exact up to one draw a border)."""
    l = np.log(np.array([0.05, 0.4, 0.25, 0.1, 0.2]))
    n = 4000
    for kw, want in (({}, [0.05, 0.4, 0.25, 0.1, 0.2]), ({"top_k": 2}, [0, 0.4, 0.25, 0, 0]),
                     ({"top_p": 0.8}, [0, 0.4, 0.25, 0, 0.2]), ({"min_p": 0.3}, [0, 0.4, 0.25, 0, 0.2]),
                     ({"top_k": 4, "top_p": 0.5}, [0, 0.4, 0.25, 0, 0])):
        got = np.bincount([F.sample_row(l, (i + 0.5) / n, **kw)[0] for i in range(n)], minlength=5)
        want = np.array(want) / sum(want)
        assert np.abs(got - n * want).max() <= 2
