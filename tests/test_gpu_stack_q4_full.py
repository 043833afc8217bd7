"""The decoder stack over a 4-bit cache when the sequences have no blocks left."""
import pytest
import torch

from fish_audio_cpp_b200 import stack as S

pytestmark = pytest.mark.gpu


@pytest.fixture
def st(ctx):
    cfg = S.SlowARConfig(n_layer=2, dim=512, n_head=4, n_kv=1, inter=512, group=64)
    st = S.SlowARStack(torch, ctx, cfg, 2, 28, max_new=4, seed=7, weight_bits=4, kv_bits=4)
    yield st
    st.close()


def tokens(st, n):
    return torch.randn((n, st.B, st.cfg.dim), generator=torch.Generator().manual_seed(2)).half().cuda()


def state(st):
    return [t.clone() for t in (st.cache4, st.block_table, st.seq_lens, st.free_count, st.free_blocks, st.out)]


def test_a_step_without_blocks_raises(st):
    room = st.max_blocks * 16 - 28
    assert st.room == room
    xs = tokens(st, room + 1)
    outs = []
    for x in xs[:room]:
        outs.append(st.decode_step(x).clone())
        st.check_plan()
    before = state(st)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="blocks"):
            st.decode_step(xs[room])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, state(st)))
    st.check_plan()
    st.reset_positions()
    assert torch.isfinite(st.decode_step(xs[0])).all()
    st.check_plan()


def test_replays_without_blocks_are_told_by_the_plan(st):
    xs = tokens(st, st.room)
    x_in = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st.decode_step(x_in)
    st.reset_positions()
    for x in xs:
        x_in.copy_(x)
        graph.replay()
        st.check_plan()
    before = state(st)[:5]
    for _ in range(2):
        graph.replay()
        with pytest.raises(RuntimeError, match="status [12]"):
            st.check_plan()
    assert all(torch.equal(a, b) for a, b in zip(before, state(st)))
    st.reset_positions()
    graph.replay()
    st.check_plan()
