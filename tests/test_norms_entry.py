"""The norms' C entries on the CPU: which calls are taken (with no rows nothing is launched) and which refused."""
import pytest

from agent_factory_3_amd import _capi

P = 4096   # an address that is never read


def _bwd(**kw):
    a = dict(dr=None, lddr=64, dh=P, lddh=64, r=P, r_f32=0, r_again=0, ldr=64, x=P, x_f32=0, ldx=64, rstd=P, rstd_x=None,
             weight=P, w_f32=0, post=None, post_f32=0, gate=None, gate_f32=0, gate_cols=0, gate_rows=1, scale=1.0,
             has_residual=0, rows=0, H=64, dx=None, dresidual=None, dweight=None, dpost=None, dgate=None, ws=None, ws_n=0,
             stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    if not _capi.lib_path().exists():
        pytest.skip("library not built")
    _capi.call("af3_residual_norm_bwd", *a.values())


def test_backward_without_a_residual_takes_either_gradient():
    """A trained weight behind a frozen x (frozen embeddings) and the other way round."""
    _bwd(dweight=P)
    _bwd(dresidual=P)
    _bwd(dresidual=P, dweight=P)
    with pytest.raises(RuntimeError, match="without a residual"):
        _bwd()
    with pytest.raises(RuntimeError, match="without a residual"):
        _bwd(dh=None, dresidual=P)
    with pytest.raises(RuntimeError, match="without a residual"):
        _bwd(dresidual=P, dx=P)


def test_workspace_does_not_grow_with_a_gates_groups():
    """A row of partials per block and sum, however many groups a gate has."""
    if not _capi.lib_path().exists():
        pytest.skip("library not built")
    size = _capi.load().af3_residual_norm_bwd_workspace_bytes
    H = 2880
    for groups in (1, 2, 100, 256, 257, 8000, 1 << 20):
        assert size(2 * groups, H, 1, H, 2, 1, 1, 1) <= 3 * 256 * H * 4, groups
