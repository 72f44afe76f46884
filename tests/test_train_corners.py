"""Corners of the training operators that need no GPU."""
import pytest
import torch

from icsa_hip import _lib, build, wan
from icsa_hip.hip_host import IcsaArgumentError

pytestmark = pytest.mark.cpu


def test_rope_positions():
    """Target, then source from 0 again; tokens behind both, and all of a grid of nothing, stay; the longest axis of either."""
    pos = wan.rope_positions([(2, 1, 2), (1, 2, 1)], [(1, 1, 3), (0, 5, 6)], 1, 2, 8, "cpu")
    assert pos.dtype == torch.int32 and pos.rope_rows == 6
    assert pos[0].tolist() == [[0, 0, 0], [0, 0, 1], [1, 0, 0], [1, 0, 1], [0, 0, 0], [0, 0, 1], [0, 0, 2], [-1, -1, -1]]
    assert pos[1].tolist() == [[0, 0, 0], [0, 1, 0]] + [[-1, -1, -1]] * 6
    assert wan.rope_positions(torch.tensor([[2, 1, 2]]), torch.tensor([[1, 1, 3]]), 0, 1, 6, "cpu")[0, 4:].tolist() == [[-1, -1, -1]] * 2
    assert wan.rope_positions([(9, 9, 9)], [(1, 1, 1)], 1, 1, 4, "cpu")[0].tolist() == [[0, 0, i] for i in range(4)]   # cut at S


@pytest.mark.parametrize("grid,src,tag", [((1, 2), (1, 2, 3), 0), ((1, 2, 3), (1, 2, 3, 4), 0), ((1, -2, 3), (1, 2, 3), 1), ((1, 2, 3), (1, 2, -3), 0),
                                          ((1, 2, 3), (1, 2, 3), 2), ((1, 2, 3), (1, 2, 3), -1)])
def test_rope_positions_refuse(grid, src, tag):
    with pytest.raises(IcsaArgumentError):
        wan.rope_positions([grid], [src], tag, 1, 8, "cpu")


@pytest.mark.parametrize("grid,src,tag", [((6, 2, 3), (1, 2, 3), 0), ((1, 2, 3), (1, 2, 9), 1), ((1, 2, 3), (1, 9, 3), 0)])
def test_a_grid_longer_than_the_table_is_refused(grid, src, tag):
    y, w, freqs = torch.zeros(1, 64, 64), torch.ones(64), wan.wan_freqs(64, 5)
    with pytest.raises(IcsaArgumentError, match="longer than the table"):
        wan.wan_qk_trainable(y, y, w, w, wan.rope_positions([grid], [src], tag, 1, 64, "cpu"), freqs, 1)


@pytest.mark.parametrize("kw,code", [
    (dict(scale=1e-30), _lib.EINVAL), (dict(q_ss=1 << 28), _lib.EUNSUPPORTED), (dict(H=8, q_sh=1 << 28), _lib.EUNSUPPORTED),
    (dict(k_ss=(1 << 24) - 64), _lib.EUNSUPPORTED), (dict(v_ss=(1 << 24) - 64), _lib.EUNSUPPORTED), (dict(q_ss=-128), _lib.EINVAL),
])
def test_the_forward_that_keeps_its_state_refuses_what_the_backward_would(kw, code):
    """At the forward's call, not after it."""
    at = 1 << 20
    a = dict(q=at, q_sb=0, q_ss=128, q_sh=128, k=at, k_sb=0, k_ss=128, k_sh=128, v=at, v_sb=0, v_ss=128, v_sh=128, B=1, Sq=8, Sk=8, H=1, Hk=1,
             D=128, qst=0, kst=0, docs=1, scale=0.1, out=at, o_sb=0, o_ss=128, o_sh=128, lse=at, rest=at, ws=0, wsb=0, stream=0)
    a.update(kw)
    assert _lib.lib().icsa_cross_attn_fwd(*a.values()) == code and _lib.lib().icsa_last_error()


def test_the_library_is_built_where_the_nodes_cannot_be(monkeypatch, tmp_path):
    """Without a host compiler: hipcc's part is linked and in place, and the failure is reported."""
    steps = []

    def run(cmd, verbose):
        steps.append(cmd)
        if cmd[0] == "no-such-compiler":
            raise RuntimeError("command failed: no-such-compiler")
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setenv("CXX", "no-such-compiler")
    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "BUILD_DIR", str(tmp_path / "objects"))
    monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "libicsa.so"))
    monkeypatch.setattr(build, "NODES_PATH", str(tmp_path / "_autograd.so"))
    with pytest.raises(RuntimeError, match="no-such-compiler"):
        build.build_library()
    assert (tmp_path / "libicsa.so").exists() and not (tmp_path / "_autograd.so").exists()
    assert sum("-shared" in cmd for cmd in steps) == 2 and len(steps) == len(build.SOURCES) + 2
