"""The decoder stack in 4 bits (weights, cache, or both) against the oracle chain, with the plan taking blocks as the sequences grow."""
import numpy as np
import pytest
import torch

from fish_audio_cpp_b200 import stack as S
from oracle import q4

pytestmark = pytest.mark.gpu


def int8_codes(ctx, w4):
    n, half = w4.shape
    w = torch.empty((n, 2 * half), dtype=torch.int8, device="cuda")
    ctx.unpack_weight4(w4, n, 2 * half, w)
    torch.cuda.synchronize()
    return w.cpu().numpy()


def pages_of(st):
    c = st.cfg
    return st.cache4.cpu().numpy().reshape(st.n_blocks, c.n_layer, st.nkv_l, q4.page_bytes(st.kv_group))


def fp16_cache(st):
    return st.k_cache.cpu().numpy().copy(), st.v_cache.cpu().numpy().copy()


def oracle_step(oracle, ctx, st, x_in, cache, table, positions, jitter=None):
    """One step on the CPU; `cache` is changed. With `jitter` the attention output moves by one fp16 ulp at random."""
    c = st.cfg
    g, D, B = c.group, c.head_dim, x_in.shape[0]
    cpu = lambda t: t.cpu().numpy()
    weight = (lambda w: int8_codes(ctx, w)) if st.weight_bits == 4 else cpu
    freqs, x, pending = cpu(st.freqs), x_in.copy(), None
    at, slot = table[np.arange(B), positions // 16], positions % 16
    for l, lw in enumerate(st.layers):
        if pending is not None:
            x = oracle.residual_add(x, pending)
        h = oracle.rms_norm(x, cpu(lw["attn_norm"]), c.eps)
        qkv = oracle.linear(weight(lw["wqkv"]), cpu(lw["sqkv"]), g, h).reshape(B, st.nq_l + 2 * st.nkv_l, D)
        norms = [cpu(lw[n]) if c.qk_norm else None for n in ("q_norm", "k_norm")]
        q, k = (np.stack([oracle.qknorm_rope(qkv[b, part], w, c.eps, freqs, int(positions[b])) for b in range(B)])
                for part, w in ((slice(0, st.nq_l), norms[0]), (slice(st.nq_l, st.nq_l + st.nkv_l), norms[1])))
        v = qkv[:, st.nq_l + st.nkv_l:]
        if st.kv_bits == 4:
            k_at, v_at, ks, vs = q4.page_places(st.kv_group)
            for b in range(B):
                page = cache[at[b], l]  # [kv heads, bytes]
                nib = np.stack([page[:, :2048] & 15, page[:, :2048] >> 4], -1).reshape(st.nkv_l, 4096)
                half = page.view(np.uint16)
                for rows, places, scale in ((k, k_at, ks), (v, v_at, vs)):
                    codes, s = q4.quantize(rows[b], st.kv_group)
                    nib[:, places[slot[b]]] = codes + 8
                    half[:, scale[slot[b], ::st.kv_group]] = s.view(np.uint16)
                page[:, :2048] = nib[:, 0::2] | nib[:, 1::2] << 4
            att, _ = q4.attention(q, cache, table, positions + 1, l, 1 / np.sqrt(D), st.kv_group)
        else:
            for x16, rows in zip(cache, (k, v)):
                x16[at, l, :, slot] = rows
            att = oracle.paged_attention_decode(q, *cache, table, positions + 1, l, 1 / np.sqrt(D))
        att16 = np.asarray(att).astype(np.float16).reshape(B, st.attn_k)
        if jitter is not None:
            bits = att16.view(np.uint16).astype(np.int32) + jitter.integers(-1, 2, att16.shape)
            att16 = np.clip(bits, 0, 0xFFFF).astype(np.uint16).view(np.float16)
        x = oracle.residual_add(x, oracle.linear(weight(lw["wo"]), cpu(lw["so"]), g, att16))
        h2 = oracle.rms_norm(x, cpu(lw["ffn_norm"]), c.eps)
        act = oracle.linear(weight(lw["w13"]), cpu(lw["s13"]), g, h2, epilogue=oracle.EPI_SWIGLU)
        pending = oracle.linear(weight(lw["w2"]), cpu(lw["s2"]), g, act)
    return oracle.rms_norm(oracle.residual_add(x, pending), cpu(st.final_norm), c.eps)


@pytest.mark.parametrize("weight_bits,kv_bits,group,kv_group,dim,context,B", [(4, 16, 64, 32, 512, 37, 3), (8, 4, 64, 32, 512, 32, 3), (4, 4, 64, 64, 512, 45, 2),
                                                                            (4, 4, 256, 32, 1024, 15, 5), (4, 4, 128, 128, 512, 0, 2)])
def test_stack_in_4_bits_matches_the_oracle_chain(ctx, oracle, weight_bits, kv_bits, group, kv_group, dim, context, B):
    """Three steps, over the border of a block; the yardstick of each is the oracle's own sensitivity to one ulp in its attention output
    (a quantiser turns a last-bit difference into another code now and then). Every step starts from the stack's own cache."""
    cfg = S.SlowARConfig(n_layer=2, dim=dim, n_head=4, n_kv=1, inter=512, group=group)
    st = S.SlowARStack(torch, ctx, cfg, B, context, max_new=40, seed=5, weight_bits=weight_bits, kv_bits=kv_bits, kv_group=kv_group)
    rng = np.random.default_rng(group + context)
    snapshot = (lambda: pages_of(st)) if kv_bits == 4 else (lambda: fp16_cache(st))
    try:
        for step in range(3):
            x_in = rng.standard_normal((B, cfg.dim)).astype(np.float16)
            before, positions = snapshot(), np.full(B, context + step)
            got = st.decode_step(torch.from_numpy(x_in).cuda()).cpu().numpy().astype(np.float32)
            ctx.check_device_status()
            table = st.block_table.cpu().numpy()
            if kv_bits == 4:
                assert st.plan_info[0].item() == 0 and st.seq_lens.tolist() == [context + step + 1] * B and st.positions.tolist() == positions.tolist()
                assert (table[:, :(context + step) // 16 + 1] >= 0).all() and (table[:, (context + step) // 16 + 1:] < 0).all()
            copy = lambda: before.copy() if kv_bits == 4 else tuple(x.copy() for x in before)
            want = oracle_step(oracle, ctx, st, x_in, copy(), table, positions).astype(np.float32)
            noise = max(np.linalg.norm(oracle_step(oracle, ctx, st, x_in, copy(), table, positions, np.random.default_rng(s)).astype(np.float32) - want)
                        for s in range(3)) / np.linalg.norm(want)
            rel = np.linalg.norm(got - want) / np.linalg.norm(want)
            assert rel < max(2e-2, 3.0 * noise), (step, rel, noise)
    finally:
        st.close()


def test_captured_steps_in_4_bits_take_blocks_as_they_go(ctx):
    """A replayed graph of one step: lengths, positions, tables and the free stack move on from replay to replay, and outputs are the eager steps' bits."""
    cfg = S.SlowARConfig(n_layer=2, dim=512, n_head=8, n_kv=2, inter=512, group=64)
    B, context, steps = 3, 30, 40
    st = S.SlowARStack(torch, ctx, cfg, B, context, max_new=64, seed=6, weight_bits=4, kv_bits=4)
    try:
        start, table0 = st.cache4.clone(), st.block_table.clone()
        xin = torch.zeros((B, cfg.dim), dtype=torch.float16, device="cuda")
        xs = torch.randn((steps, B, cfg.dim), generator=torch.Generator().manual_seed(1)).half().cuda()

        def again():
            st.reset_positions()
            st.cache4.copy_(start)
            st.block_table.copy_(table0)

        eager = []
        for x in xs:
            eager.append(st.decode_step(x).clone())
        table = st.block_table.clone()
        again()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st.decode_step(xin)
        again()
        for x, want in zip(xs, eager):
            xin.copy_(x)
            graph.replay()
            assert torch.equal(st.out, want)
        assert torch.equal(st.block_table, table) and st.seq_lens.tolist() == [context + steps] * B
        assert st.free_count.item() == st.free0 - B * ((context + steps + 15) // 16 - (context + 15) // 16)
        ctx.check_device_status()
    finally:
        st.close()


def test_stack_refuses_4_bits_across_gpus(ctx):
    with pytest.raises(AssertionError, match="one GPU"):
        S.SlowARStack(torch, ctx, S.SlowARConfig(n_layer=1), 1, 0, tp_size=2, weight_bits=4)
