"""CPU checks of the decay-attention and beam-search entry points: refusals without a GPU and through the C ABI."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from gla_jax_b200 import build, _lib
    build.build()
    return _lib.load()


def test_cpu_tensors_raise():
    import gla_jax_b200 as g
    h, x = torch.zeros(1, 2, 8, 8), torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        g.chunk_decay_attention(h, x[..., 0], x, x, x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        g.chunk_decay_attention_packed(h, x[0, ..., 0], x[0], x[0], x[0], [0, 4])
    with pytest.raises(ValueError, match="rise"):
        g.chunk_decay_attention_packed(h, x[0, ..., 0], x[0], x[0], x[0], [0, 5])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        g.decay_attention_step(h, x[:, 0, :, 0], x[:, 0], x[:, 0], x[:, 0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        g.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        g.reorder_states([h], torch.zeros(1, 1, dtype=torch.int32))


def test_validation_without_gpu(lib):
    """Bad arguments are turned down before anything is launched, so these calls are safe on a CPU box."""
    p, odd, big = ctypes.c_void_p(4096), ctypes.c_void_p(4100), 1 << 40
    fwd = lambda B, T, H, Hk, Dk, Dv, dt=1, hdt=1, nseq=0, cu=None, h=p, v=p, ws=p, n=big: lib.gla_decay_fwd(  # noqa: E731
        None, B, T, H, Hk, Dk, Dv, dt, hdt, nseq, cu, h, p, 1, v, p, p, p, p, None, ws, n)
    assert fwd(1, 8, 2, 2, 64, 64, h=None) == 1
    assert fwd(0, 8, 2, 2, 64, 64) == fwd(1, 0, 2, 2, 64, 64) == fwd(1, 8, 3, 2, 64, 64) == 2
    assert fwd(2, 8, 2, 2, 64, 64, nseq=1, cu=p) == fwd(1, 8, 2, 2, 64, 64, nseq=1) == fwd(1, 8, 2, 2, 64, 64, cu=p) == 2
    assert fwd(1, 8, 2, 2, 60, 64) == fwd(1, 8, 2, 2, 264, 64) == fwd(1, 8, 2, 2, 64, 64, dt=7) == fwd(1, 8, 2, 2, 64, 64, dt=0, hdt=1) == 3
    assert fwd(1, 8, 2, 2, 64, 64, v=odd) == 4
    assert lib.gla_decay_workspace_bytes(1, 8, 2, 2, 64, 64, 1, 1, 0, 0) == 0
    need = lib.gla_decay_workspace_bytes(1, 65536, 2, 2, 64, 64, 1, 1, 0, 0)
    assert need > 0 and fwd(1, 65536, 2, 2, 64, 64, n=need - 1) == fwd(1, 65536, 2, 2, 64, 64, ws=None) == 5
    assert lib.gla_decay_workspace_bytes(1, 65536, 2, 1, 64, 64, 1, 1, 0, 3) > lib.gla_decay_workspace_bytes(1, 65536, 2, 2, 64, 64, 1, 1, 0, 2) > 0
    assert lib.gla_decay_saved_bytes(1, 8, 2, 2, 64, 64, 1, 1, 0) >= 2 * 64 * 64 * 4 and lib.gla_decay_saved_bytes(1, 8, 3, 2, 64, 64, 1, 1, 0) == 0
    assert lib.gla_decay_workspace_bytes(1, 8, 2, 2, 60, 64, 1, 1, 0, 0) == 0
    step = lambda B=4, Dk=64, parents=None, beams=1, state=p: lib.gla_decay_step(  # noqa: E731
        None, B, 2, 2, Dk, 64, 1, state, p, p, p, p, p, 1, parents, beams)
    assert step(state=None) == 1 and step(B=0) == 2 and step(parents=p, beams=3) == 2 and step(Dk=12) == 3 and step(state=odd) == 4
    assert step(B=33, parents=p, beams=33) == 3
    assert lib.gla_decode_step_beams(None, 4, 2, 48, 1, p, p, p, p, p, p, 1, p, 2) == 3
    assert lib.gla_decode_step_beams(None, 4, 2, 64, 1, p, p, p, p, p, p, 1, None, 2) == 1
    sel = lambda N=1, K=2, V=9, M=2, pad=0, x=p, ws=p, n=big: lib.gla_beam_select(  # noqa: E731
        None, N, K, V, M, 0, x, p, None, pad, p, p, p, ws, n)
    assert sel(x=None) == 1 and sel(M=19) == 2 and sel(pad=9) == 2 and sel(K=33) == 3 and sel(M=33, V=99) == 3
    assert sel(x=ctypes.c_void_p(4098)) == 4 and sel(n=8) == 5
    assert lib.gla_beam_select_workspace_bytes(1, 2, 9, 19, 0) == 0 < lib.gla_beam_select_workspace_bytes(1, 2, 9, 2, 0)
    assert lib.gla_reorder_states(None, 0, p, p, 1, 2, p) == 0
    assert lib.gla_reorder_states(None, 1, None, p, 1, 2, p) == 1
    assert lib.gla_reorder_states(None, 0, p, p, 1, 33, p) == 3


def test_no_states_to_move(lib):
    """An empty list has no arrays behind it: there is nothing to do, which is no error."""
    p = ctypes.c_void_p(4096)
    assert lib.gla_reorder_states(None, 0, None, None, 2, 4, p) == 0
    assert lib.gla_reorder_states(None, 0, None, None, 2, 4, None) == 1
    assert lib.gla_reorder_states(None, 1, p, None, 2, 4, p) == 1


def test_what_a_packed_call_and_a_backward_keep(lib):
    """Offsets travel in the workspace of a forward alone and in `saved` of one that is differentiated; what has no other state to
    keep (float32, head sizes beyond 128) may go without `saved`."""
    p, big = ctypes.c_void_p(4096), 1 << 40
    ws = lambda *a: lib.gla_decay_workspace_bytes(*a)  # noqa: E731
    assert ws(1, 8, 2, 2, 64, 64, 1, 1, 3, 0) >= 16 and ws(1, 8, 2, 2, 64, 64, 1, 1, 3, 1) == 0
    assert lib.gla_decay_saved_bytes(1, 8, 2, 2, 64, 64, 0, 0, 0) == lib.gla_decay_saved_bytes(1, 8, 2, 2, 256, 64, 1, 1, 0) == 0
    assert lib.gla_decay_saved_bytes(1, 8, 2, 2, 64, 64, 0, 0, 3) >= 16
    assert lib.gla_decay_saved_bytes(1, 8, 2, 2, 64, 64, 1, 1, 3) >= 3 * 2 * 64 * 64 * 4 + 16
    assert ws(1, 8, 2, 2, 64, 64, 0, 0, 0, 3) >= 2 * 64 * 64 * 4 + ws(1, 8, 2, 2, 64, 64, 0, 0, 0, 2)
    bwd = lambda dt, nseq, cu, saved, n=big: lib.gla_decay_bwd(  # noqa: E731
        None, 1, 8, 2, 2, 64, 64, dt, dt, nseq, cu, p, p, 1, p, p, p, saved, p, p, p, p, p, p, p, p, n)
    assert bwd(1, 0, None, None) == 1 and bwd(0, 1, p, None) == 1
    assert bwd(0, 0, None, None, 16) == 5 and bwd(1, 0, None, ctypes.c_void_p(4100)) == 4
    step = lambda B, H, parents=None, beams=1: lib.gla_decay_step(None, B, H, H, 64, 64, 1, None, p, p, p, p, p, 1, parents, beams)  # noqa: E731
    assert step(1 << 20, 16) == 1                    # (a null state is all that is wrong)
    sizes = lambda B, H: lib.gla_decay_step(None, B, H, H, 64, 64, 1, p, p, p, p, p, p, 1, None, 1)  # noqa: E731
    assert sizes(1 << 32, 1) == sizes(1 << 22, 16) == 8
