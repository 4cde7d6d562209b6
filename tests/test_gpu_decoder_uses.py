"""The decoder operators as programs use them: several layers in a plan, captured graphs, other streams, launches without overlap, sizes
whose offsets pass 32 bits. The results are those of the plain use, bit for bit, which test_gpu_decoder_ops.py holds against the oracle."""
import numpy as np
import pytest

from oracle import decoder as D
from snntome_b200.native import KV8Cache, NativeError, NativePlan

pytestmark = pytest.mark.gpu


def random_canvas(plan, rows, pitch, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    canvas = plan.canvas_tensor()
    for r in range(0, rows, 4096):
        n = min(4096, rows - r) * pitch
        canvas[r * pitch: r * pitch + n] = torch.randn(n, generator=g, device="cuda", dtype=torch.float32).to(torch.float16)
    return canvas


def loaded_cache(columns, h_kv, dim, max_seq, seed):
    """A cache whose first three blocks of every column and head, and open blocks, hold something."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = KV8Cache(columns, h_kv, dim, max_seq)
    v = cache.views()
    codes = v["codes"].view(torch.uint8)[:, :, :3]
    codes.copy_(torch.randint(0, 120, codes.shape, generator=g, device="cuda", dtype=torch.uint8))
    v["scales"][:, :, :3] = 0.01
    for part in ("k_tail", "v_tail"):
        v[part].copy_(torch.randn(v[part].shape, generator=g, device="cuda").to(torch.float16))
    v["tail_block"].fill_(1)
    return cache


def attention(plan, cache, pitch, row, h_q, **kw):
    rq, rk = h_q * cache.head_dim, cache.h_kv * cache.head_dim
    plan.add_kv8_attn(cache, row * pitch, (row + rq) * pitch, (row + rq + rk) * pitch, (row + rq + 2 * rk) * pitch, h_q, **kw)
    return row + 2 * rq + 2 * rk


POSITIONS = np.array([70, 100, -1, 127, 64, 90, 0, 127], dtype=np.int32)
LAYERS = [(4, 2, 64, 0), (16, 1, 128, 40), (8, 1, 64, 0)]          # query heads, key / value heads, dimensions, window: scratch grows from one to the next


def layers(how):
    """Runs three layers over caches of their own and returns the canvas behind them and the caches' bytes."""
    import torch
    columns, pitch = POSITIONS.size, 64
    rows = sum(2 * q * d + 2 * k * d for q, k, d, _ in LAYERS)
    plan = NativePlan.create(rows * pitch, pitch, columns)
    canvas = random_canvas(plan, rows, pitch, 3)
    start = canvas.clone()
    caches = [loaded_cache(columns, k, d, 200, i) for i, (q, k, d, w) in enumerate(LAYERS)]
    row, between = 0, [c.storage.clone() for c in caches]
    for (q, k, d, w), cache in zip(LAYERS, caches):
        row = attention(plan, cache, pitch, row, q, window=w, sinks=2)
        if how == "grown":                                          # run and captured before the next layer's scratch is made
            plan.set_positions(POSITIONS)
            plan.execute()
            plan.execute_graph()
    for c, b in zip(caches, between):
        c.storage.copy_(b)
    canvas.copy_(start)
    if how == "side stream":
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        plan.set_positions(POSITIONS, stream=s)
        plan.execute(stream=s)
        s.synchronize()
    elif how == "captured":
        plan.set_positions(POSITIONS)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            plan.execute(stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        g.replay()
        g.replay()                                                  # the same token again
        torch.cuda.synchronize()
        del g
    elif how == "grown":
        plan.execute_graph()
    else:
        plan.set_positions(POSITIONS)
        plan.execute()
    assert plan.status() == 0
    out = canvas.clone(), [c.storage.clone() for c in caches]
    plan.close()
    return out


@pytest.mark.parametrize("how", ["side stream", "captured", "grown", "no overlap"])
def test_layers_of_one_plan(how, monkeypatch):
    import torch
    want, kept = layers("plain")
    if how == "no overlap":
        monkeypatch.setenv("K44B_PDL", "0")
    got, left = layers(how)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    for a, b in zip(left, kept):
        assert torch.equal(a, b)


def test_a_layer_that_cannot_be_added_leaves_the_others():
    import torch
    columns, pitch = POSITIONS.size, 64
    plan = NativePlan.create(4096 * pitch, pitch, columns)
    canvas = random_canvas(plan, 4096, pitch, 4)
    cache = loaded_cache(columns, 2, 64, 200, 5)
    row = attention(plan, cache, pitch, 0, 4)
    plan.set_positions(POSITIONS)
    plan.execute_graph()
    want = canvas.clone()
    for bad in [dict(h_q=32), dict(h_q=3)]:
        with pytest.raises(NativeError):
            attention(plan, cache, pitch, 4000, **bad)
    with pytest.raises(NativeError):
        plan.add_window_attn(0, 0, 0, 0, 1, 1, 64, 1)
    plan.execute_graph()
    assert plan.status() == 0
    assert torch.equal(canvas.view(torch.int16), want.view(torch.int16))
    plan.close()


def test_two_plans_take_turns_in_one_captured_graph():
    """A prompt's attention and the filling of the cache, and a token's attention to it, captured together and replayed on changed inputs."""
    import torch
    h_q, h_kv, dim, seq, frames = 4, 2, 64, 77, 3
    rq, rk = h_q * dim, h_kv * dim

    def build():
        pitch = 256
        prompt = NativePlan.create((2 * rq + 2 * rk) * pitch, pitch, frames * seq)
        pc = random_canvas(prompt, 2 * rq + 2 * rk, pitch, 7)
        cache = KV8Cache(frames, h_kv, dim, 128)
        prompt.add_window_attn(0, rq * pitch, (rq + rk) * pitch, (rq + 2 * rk) * pitch, h_q, h_kv, dim, seq, window=30, sinks=1)
        prompt.add_kv8_fill(cache, rq * pitch, (rq + rk) * pitch, seq)
        prompt.set_sequences([2, 1, 0], [77, 64, 5])
        token = NativePlan.create((2 * rq + 2 * rk) * 64, 64, frames)
        tc = random_canvas(token, 2 * rq + 2 * rk, 64, 8)
        attention(token, cache, 64, 0, h_q, window=30, sinks=1)
        token.set_positions([5, 64, 77])
        torch.cuda.synchronize()
        return prompt, pc, cache, token, tc

    def inputs(pc, tc):
        pc[: (rq + 2 * rk) * 256] = -pc[: (rq + 2 * rk) * 256].flip(0)
        tc[: (rq + 2 * rk) * 64] = tc[: (rq + 2 * rk) * 64].flip(0)

    prompt, pc, cache, token, tc = build()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        prompt.execute(stream=s)
        token.execute(stream=s)
    for _ in range(2):
        inputs(pc, tc)
        g.replay()
    torch.cuda.synchronize()
    got = pc.clone(), tc.clone(), cache.storage.clone()
    assert prompt.status() == 0 and token.status() == 0
    del g
    prompt.close(), token.close()
    prompt, pc, cache, token, tc = build()
    for _ in range(2):
        inputs(pc, tc)
        prompt.execute()
        token.execute()
    torch.cuda.synchronize()
    for a, b in zip(got, (pc, tc, cache.storage)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    prompt.close(), token.close()


def test_a_sequence_may_be_all_of_the_plan():
    """seq_len is a bound: one far beyond the plan's columns does what the columns' number does."""
    import torch
    got = []
    for seq in (100, (1 << 31) - 1):
        cache = KV8Cache(1, 2, 64, 90)
        plan = NativePlan.create(12 * 64 * 128, 128, 100)
        canvas = random_canvas(plan, 8 * 64, 128, 23)
        plan.add_kv8_fill(cache, 4 * 64 * 128, 6 * 64 * 128, seq)
        plan.add_window_attn(0, 4 * 64 * 128, 6 * 64 * 128, 8 * 64 * 128, 4, 2, 64, seq, window=(1 << 31) - 1, sinks=(1 << 31) - 1)
        plan.set_sequences([0], [90])
        plan.execute()
        assert plan.status() == 0
        # Not the same bits: a warp moves its columns' maxima together, those behind the plan's last one too, and they see other keys.
        x = canvas.cpu().numpy().reshape(-1, 128)[:, :100]
        y = x[: 8 * 64].astype(np.float64)
        want, bound = D.window_attention(y[: 4 * 64], y[4 * 64: 6 * 64], y[6 * 64:], 4, 2, 100, 100, 0, 0, 10000.0)
        assert np.all(np.abs(x[8 * 64:] - want) <= bound)
        got.append(cache.storage.clone())
        plan.close()
    assert torch.equal(got[0], got[1])


def test_cache_beyond_32_bits():
    """Codes of the last columns lie more than 4 GiB into the cache; a cache of short columns does the same arithmetic."""
    import torch
    columns, h_kv, dim, h_q, pitch = 70, 8, 128, 16, 128
    rq, rk = h_q * dim, h_kv * dim
    got = []
    for max_seq in (192, 32768):
        plan = NativePlan.create((2 * rq + 2 * rk) * pitch, pitch, columns)
        canvas = random_canvas(plan, 2 * rq + 2 * rk, pitch, 11)
        cache = loaded_cache(columns, h_kv, dim, max_seq, 12)
        assert max_seq == 192 or cache.storage.numel() > 1 << 32
        v = cache.views()
        attention(plan, cache, pitch, 0, h_q)
        positions = np.full(columns, -1, dtype=np.int32)
        positions[[0, 34, 68, 69]] = [3, 127, 100, 127]
        plan.set_positions(positions)
        plan.execute()
        assert plan.status() == 0
        fill = NativePlan.create(2 * rk * 192, 192, 190)
        random_canvas(fill, 2 * rk, 192, 13)
        fill.add_kv8_fill(cache, 0, rk * 192, 95)
        fill.set_sequences([66, 67], [95, 64])
        fill.execute()
        assert fill.status() == 0
        got.append([canvas.clone()] + [v[part][:, :, :3].contiguous() if part in ("codes", "scales") else v[part].clone() for part in ("codes", "scales", "k_tail", "v_tail", "tail_block")])
        plan.close(), fill.close()
        del cache, v
    for a, b in zip(*got):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_prompt_beyond_32_bits():
    """The last head's q and output lie more than 2^31 elements into the canvas; a plan of that head alone does the same arithmetic."""
    import torch
    h_q, dim, seq, window = 130, 128, 131072, 64
    pitch, rq = seq, h_q * dim
    plan = NativePlan.create((2 * rq + 2 * dim) * pitch, pitch, seq)
    canvas = random_canvas(plan, rq + 2 * dim, pitch, 17)
    plan.add_window_attn(0, rq * pitch, (rq + dim) * pitch, (rq + 2 * dim) * pitch, h_q, 1, dim, seq, window=window, sinks=3)
    plan.execute()
    assert plan.status() == 0
    one = NativePlan.create(4 * dim * pitch, pitch, seq)
    alone = one.canvas_tensor()
    alone[: 3 * dim * pitch] = canvas[(rq - dim) * pitch: (rq + 2 * dim) * pitch]
    one.add_window_attn(0, dim * pitch, 2 * dim * pitch, 3 * dim * pitch, 1, 1, dim, seq, window=window, sinks=3)
    one.execute()
    assert one.status() == 0
    assert torch.equal(canvas[-dim * pitch:].view(torch.int16), alone[-dim * pitch:].view(torch.int16))
    plan.close(), one.close()


def test_logits_beyond_32_bits():
    import torch
    rows, columns, top = 131072, 16448, 3
    plan = NativePlan.create(rows * columns, columns, columns)
    canvas = random_canvas(plan, rows, columns, 19)
    assert canvas.numel() > 1 << 31
    targets = torch.full((columns,), rows - 1, dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(columns, device="cuda"), torch.empty(columns, device="cuda")
    tr, tl = torch.empty(top, columns, dtype=torch.int32, device="cuda"), torch.empty(top, columns, device="cuda")
    plan.add_logprobs(0, rows, targets, lp, ent, tr, tl)
    plan.execute()
    assert plan.status() == 0
    for c in (0, 8191, columns - 1):
        x = canvas.view(rows, columns)[:, c].double()
        p = torch.log_softmax(x, 0)
        # a 32-bit result of magnitude 12, sums of 2^17 terms in a tree: see the oracle's tests for the bound
        assert abs(lp[c].item() - p[-1].item()) <= 2.0 ** -21 * abs(p[-1].item()) + 8e-6
        assert abs(ent[c].item() + (p.exp() * p).sum().item()) <= 2.0 ** -20 * 12 + 8e-6
        order = torch.argsort(x, descending=True, stable=True)[:top]
        assert torch.equal(tr[:, c].long(), order)
        assert (tl[:, c].double() - p[order]).abs().max().item() <= 2.0 ** -21 * 12 + 8e-6
    plan.close()
