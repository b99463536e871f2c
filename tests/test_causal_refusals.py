"""What the causal mixer's C entry points and modules refuse before anything is launched, without a GPU."""
import ctypes

import pytest
import torch


def _p(address=4096):
    return ctypes.c_void_p(address)


def _scan(lib_mod, **changes):
    s = lib_mod.ScanInputs()
    for f in ("x", "dt", "Bm", "Cm", "A"):
        setattr(s, f, 4096)
    s.batch, s.length, s.channels, s.groups, s.states = 2, 8, 16, 1, 4
    for k, v in changes.items():
        setattr(s, k, v)
    return ctypes.byref(s)


def test_conv_entry_points():
    from m2_amd._lib import lib
    ok = _p()

    def fwd(x=ok, w=ok, y=ok, B=1, L=8, C=16, K=4, dtype=0):
        return lib.m2_causal_conv_fwd(x, 128, 16, w, None, None, None, y, None, B, L, C, K, 0, dtype, None)

    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(y=None) == -1 and b"null" in lib.m2_last_error()
    assert fwd(B=0) == -1 and fwd(L=0) == -1 and fwd(C=0) == -1 and fwd(B=65536) == -1 and fwd(dtype=2) == -1
    assert fwd(K=0) == -2 and fwd(K=9) == -2 and b"9 taps" in lib.m2_last_error()
    assert fwd(C=(1 << 20) + 1) == -1 and fwd(L=(1 << 30) + 1) == -1 and fwd(B=65535, L=1 << 20, C=1 << 10) == -1 and b"2^36" in lib.m2_last_error()

    def bwd(gy=ok, workspace=ok, gw=ok, K=4):
        return lib.m2_causal_conv_bwd(ok, 128, 16, ok, None, None, None, gy, 128, 16, None, ok, gw, None, None, workspace, 1, 8, 16, K, 0, 0, None)

    assert bwd(gy=None) == -1 and bwd(workspace=None) == -1 and bwd(K=9) == -2
    assert lib.m2_causal_conv_bwd_workspace_bytes(1, 8, 16, 9, 0) == 0 and lib.m2_causal_conv_bwd_workspace_bytes(1, 8, 16, 4, 0) >= 4 * 5 * 16
    assert lib.m2_causal_conv_step(ok, 16, None, ok, None, ok, ok, 1, 16, 4, 0, 0, None) == -1
    assert lib.m2_causal_conv_step(ok, 16, ok, ok, None, ok, ok, 65535, 1 << 20, 4, 0, 0, None) == -1


def test_scan_entry_points():
    from m2_amd import _lib
    from m2_amd._lib import lib

    def fwd(y=_p(), dtype=0, **changes):
        return lib.m2_selective_scan_fwd(_scan(_lib, **changes), y, None, None, dtype, None)

    assert lib.m2_selective_scan_fwd(None, _p(), None, None, 0, None) == -1 and fwd(y=None) == -1
    for f in ("x", "dt", "Bm", "Cm", "A"):
        assert fwd(**{f: None}) == -1 and b"null" in lib.m2_last_error()
    assert fwd(batch=0) == -1 and fwd(length=0) == -1 and fwd(channels=0) == -1 and fwd(groups=3) == -1 and fwd(groups=0) == -1 and fwd(dtype=5) == -1
    assert fwd(states=0) == -2 and fwd(states=257) == -2 and b"257 states" in lib.m2_last_error()
    assert fwd(channels=(1 << 20) + 1) == -1 and fwd(batch=1 << 20, channels=128) == -1 and fwd(length=1 << 30, batch=32) == -1
    g = _lib.ScanGradients()
    assert lib.m2_selective_scan_bwd(_scan(_lib), ctypes.byref(g), _p(), _p(), 0, None) == -1      # no gy
    g.gy = 4096
    assert lib.m2_selective_scan_bwd(_scan(_lib), ctypes.byref(g), None, _p(), 0, None) == -1
    assert lib.m2_selective_scan_bwd(_scan(_lib), ctypes.byref(g), _p(), None, 0, None) == -1
    assert lib.m2_selective_scan_bwd(_scan(_lib), None, _p(), _p(), 0, None) == -1
    assert lib.m2_selective_scan_step(_scan(_lib, length=1), _p(), _p(), 0, None) == -1      # no state
    assert lib.m2_selective_scan_step(_scan(_lib, length=1, state=4096), _p(), None, 0, None) == -1
    assert lib.m2_selective_scan_step(_scan(_lib, length=1, state=4096, batch=1 << 20, channels=64, states=256), _p(), _p(), 0, None) == -1 and b"launch" in lib.m2_last_error()
    assert fwd(batch=1 << 20, channels=64, states=256) == -1 and b"launch" in lib.m2_last_error()
    for row in ("x_row", "dt_row", "z_row", "b_row", "c_row"):
        assert fwd(**{row: 1 << 24}) == -2 and fwd(**{row: -1}) == -2 and b"2^24" in lib.m2_last_error()
    assert [lib.m2_selective_scan_span(n) for n in (0, 257)] == [0, 0]
    for n in (1, 16, 64, 100, 256):
        assert lib.m2_selective_scan_span(n) % 16 == 0 and lib.m2_selective_scan_span(n) >= 32
    assert lib.m2_selective_scan_bwd_workspace_bytes(2, 8, 16, 1, 300) == 0
    # partial gradients of B and C, one of each from a workgroup at least, and of A, D and dt_bias for each sequence
    assert lib.m2_selective_scan_bwd_workspace_bytes(2, 8, 16, 1, 4) >= 4 * (2 * 2 * 8 * 4 + 2 * 16 * 4 + 2 * 2 * 16)


def test_norm_entry_points():
    from m2_amd._lib import lib
    ok = _p()

    def fwd(x=ok, y=ok, stats=ok, workspace=ok, N=2, S=3, C=16, G=4, act=0, dtype=0):
        return lib.m2_group_norm_fwd(x, S * C, C, None, None, 1e-5, y, stats, workspace, N, S, C, G, act, dtype, None)

    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(stats=None) == -1 and fwd(workspace=None) == -1 and b"workspace" in lib.m2_last_error()
    assert fwd(N=0) == -1 and fwd(S=0) == -1 and fwd(C=0) == -1 and fwd(G=3) == -1 and fwd(G=0) == -1 and fwd(act=3) == -1 and fwd(dtype=-1) == -1
    assert fwd(N=1 << 24) == -1 and fwd(N=1 << 31) == -1
    assert lib.m2_group_norm_bwd(ok, 48, 16, None, None, None, ok, 48, 16, ok, None, None, ok, 2, 3, 16, 4, 0, 0, None) == -1
    assert lib.m2_group_norm_bwd(ok, 48, 16, None, None, ok, ok, 48, 16, ok, ok, None, None, 2, 3, 16, 4, 0, 0, None) == -1
    assert lib.m2_group_norm_workspace_bytes(2, 1, 16, 4, 0, 0) == 0 and lib.m2_group_norm_workspace_bytes(2, 3, 16, 4, 0, 0) > 0
    assert lib.m2_group_norm_workspace_bytes(2, 3, 16, 5, 0, 0) == 0


def test_modules_refuse_what_is_not_on_the_gpu():
    import m2_amd
    x, w, s = torch.randn(2, 5, 8), torch.randn(8, 4), torch.randn(2, 3, 8)
    A, B = -torch.ones(8, 4), torch.randn(2, 5, 4)
    calls = [lambda: m2_amd.causal_conv(x, w), lambda: m2_amd.causal_conv_step(x[:, 0], s, w), lambda: m2_amd.selective_scan(x, x, A, B, B),
             lambda: m2_amd.selective_scan_step(x[:, 0], x[:, 0], torch.zeros(2, 8, 4), A, B[:, 0], B[:, 0]), lambda: m2_amd.group_norm(x, 4)]
    for call in calls:
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    for activation in ("relu", "SiLU", 1):
        with pytest.raises(ValueError, match="activation"):
            m2_amd.causal_conv(x, w, activation=activation)
        with pytest.raises(ValueError, match="activation"):
            m2_amd.group_norm(x, 4, activation=activation)
    with pytest.raises(ValueError):
        m2_amd.causal_conv(x, w, activation="gelu")
    with pytest.raises(TypeError):
        m2_amd.causal_conv(None, w)
    with pytest.raises(TypeError):
        m2_amd.group_norm([[1.0]], 1)


def test_without_their_extension_only_they_raise():
    import os
    import subprocess
    import sys
    code = ("import sys, warnings\n"
            "sys.modules['m2_amd._causal_calls'] = None\n"
            "with warnings.catch_warnings(record=True) as seen:\n"
            "    warnings.simplefilter('always')\n"
            "    import m2_amd\n"
            "assert any('_causal_calls' in str(w.message) and 'build' in str(w.message) for w in seen)\n"
            "import torch\n"
            "x = torch.ones(1, 2, 4)\n"
            "for call in (lambda: m2_amd.causal_conv(x, torch.ones(4, 2)), lambda: m2_amd.group_norm(x, 2), lambda: m2_amd.selective_scan(x, x, x[0], x, x)):\n"
            "    try:\n"
            "        call()\n"
            "    except RuntimeError as e:\n"
            "        assert 'build' in str(e)\n"
            "    else:\n"
            "        raise AssertionError\n"
            "cfg = m2_amd.m2_bert_80m(128)\n"
            "cfg.num_hidden_layers = 1\n"
            "m2_amd.BertModel(cfg)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_scan_gradient_workspace_stays_in_proportion():
    """Partial gradients of B and C: 1 GiB, or sixteen bytes for each value of x; sets of channels share one where there would be more, as far as shared memory holds them (29 channels of 65 to 128 states)."""
    from m2_amd._lib import lib
    for batch, length, channels, groups, states in ((8, 2048, 1536, 1, 16), (8, 2048, 1536, 1, 128), (1, 131072, 1536, 1, 16), (4, 4096, 4096, 8, 64), (8, 2048, 3584, 1, 100)):
        rest = 4 * (batch * channels * (states + 2))
        assert lib.m2_selective_scan_bwd_workspace_bytes(batch, length, channels, groups, states) <= max(1 << 30, 16 * batch * length * channels, 8 * batch * length * states * -(-channels // 29)) + rest, (batch, length, channels, groups, states)
