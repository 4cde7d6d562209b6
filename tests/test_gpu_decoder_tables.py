"""The tables that the decoder operators read (positions, sequences), their scratch under captured graphs, and positions at the ends of a
cache and of its blocks."""
import numpy as np
import pytest

import test_gpu_decoder_ops as ops
from oracle import decoder as D
from snntome_b200.native import KV8Cache, NativeError, NativePlan

pytestmark = pytest.mark.gpu


def busy_default_stream():
    """Some tens of milliseconds of work on the default stream, and a stream that does not wait for it."""
    import torch
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    torch.cuda._sleep(100_000_000)
    return s


def test_positions_set_before_the_command_on_a_stream_of_their_own():
    import torch
    h_q, h_kv, dim = 2, 1, 64
    pitch = 64
    rng = np.random.default_rng(1)
    body = rng.normal(0, 1, (4 * dim, pitch)).astype(np.float16)
    out = []
    for early in (False, True):
        plan, canvas = ops.make_plan(body, 2 * dim, 3)
        cache = KV8Cache(3, h_kv, dim, 100)
        torch.cuda.synchronize()
        s = torch.cuda.current_stream()
        if early:
            s = busy_default_stream()
            plan.set_positions([0, -1, 0], stream=s)
        plan.add_kv8_attn(cache, 0, 2 * dim * pitch, 3 * dim * pitch, 4 * dim * pitch, h_q)
        if not early:
            plan.set_positions([0, -1, 0])
        plan.execute(stream=s)
        assert plan.status() == 0
        out.append(ops.read(canvas, pitch)[4 * dim:, :3].copy())
        plan.close()
    assert out[0][:, 0].any() and np.array_equal(out[0].view(np.uint16), out[1].view(np.uint16))


@pytest.mark.parametrize("first", ["table", "command"])
def test_sequences_set_on_a_stream_of_their_own(first):
    import torch
    h_kv, dim, seq = 2, 64, 70
    rk, pitch = h_kv * dim, 256
    body = np.random.default_rng(2).normal(0, 1, (2 * rk, pitch)).astype(np.float16)
    plan, canvas = ops.make_plan(body, rk, 3 * seq)
    plan.add_window_attn(0, 0, rk * pitch, 2 * rk * pitch, h_kv, h_kv, dim, seq)          # its angles are those of the filling too
    cache = KV8Cache(4, h_kv, dim, 100)
    if first == "table":
        s = busy_default_stream()
        plan.set_sequences([3, -1, 0], [70, 70, 64], stream=s)
        plan.add_kv8_fill(cache, 0, rk * pitch, seq)
    else:
        s = busy_default_stream()
        plan.add_kv8_fill(cache, 0, rk * pitch, seq)
        plan.set_sequences([3, -1, 0], [70, 70, 64], stream=s)
    plan.execute(stream=s)
    assert plan.status() == 0
    a = ops.cache_arrays(cache)
    assert a["tail_block"].tolist() == [[-1, -1], [-1, -1], [-1, -1], [1, 1]] and (a["scales"][[0, 3], :, 0] > 0).all()
    plan.close()


def test_a_plan_made_and_used_while_the_default_stream_is_busy():
    """Its canvas is clear when the call returns, so that what other streams write then stays."""
    import torch
    body = torch.randn(8 * 64, 64, device="cuda").to(torch.float16)
    out = []
    for busy in (False, True):
        s = busy_default_stream() if busy else torch.cuda.Stream()
        plan = NativePlan.create(14 * 64 * 64, 64, 50)
        with torch.cuda.stream(s):
            canvas = plan.canvas_tensor()
            canvas[: body.numel()].copy_(body.reshape(-1))
            plan.add_window_attn(0, 2 * 64 * 64, 3 * 64 * 64, 8 * 64 * 64, 2, 1, 64, 50)
            plan.execute(stream=s)
        assert plan.status() == 0
        out.append(canvas.clone())
        plan.close()
    assert bool(out[0][8 * 64 * 64:].any()) and torch.equal(out[0], out[1])


def test_a_captured_graph_keeps_its_scratch_when_commands_are_added():
    """Captured by the caller, then larger commands of every kind; what the graph holds must not be given to others meanwhile."""
    import torch
    h_q, h_kv, dim, pitch, columns, rows = 4, 2, 64, 64, 40, 1000
    rq, rk = h_q * dim, h_kv * dim
    rng = np.random.default_rng(3)
    body = rng.normal(0, 1, (rq + 2 * rk + rows, pitch)).astype(np.float16)
    plan, canvas = ops.make_plan(body, 2 * rq + 8192, columns)
    out, late = (rq + 2 * rk + rows) * pitch, (2 * rq + rq + 2 * rk + rows) * pitch
    cache = KV8Cache(columns, h_kv, dim, 400)
    cache.storage[: cache.storage.numel() // 2] = 20
    cache.views()["scales"].fill_(0.01)
    cache.views()["tail_block"].fill_(4)
    plan.add_window_attn(0, rq * pitch, (rq + rk) * pitch, out, h_q, h_kv, dim, 20, window=5)
    plan.add_kv8_attn(cache, 0, rq * pitch, (rq + rk) * pitch, out + rq * pitch, h_q)
    f = lambda *s: torch.zeros(s, device="cuda")
    ent, rows_t, lp_t = f(columns), torch.zeros(3, columns, dtype=torch.int32, device="cuda"), f(3, columns)
    plan.add_logprobs((rq + 2 * rk) * pitch, rows, entropy=ent, top_rows=rows_t, top_logprobs=lp_t)
    plan.add_argmax((rq + 2 * rk) * pitch, rows)
    plan.set_positions(np.full(columns, 300))
    plan.execute()
    assert plan.status() == 0
    want = [canvas[out: late].clone(), ent.clone(), rows_t.clone(), lp_t.clone(), plan.next_tokens(columns)]
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        plan.execute(stream=s)
    # larger ones: more heads, wider groups, more rows
    plan.add_window_attn(0, 0, 0, late, 4, 4, 64, 20)
    for heads, kv, d in ((5, 1, 128), (9, 1, 128), (4, 4, 64)):
        plan.add_kv8_attn(KV8Cache(columns, kv, d, 400), 0, 0, 0, late, heads)
    plan.add_logprobs(0, 6000, entropy=f(columns))
    plan.add_argmax(0, 6000)
    torch.cuda.synchronize()
    taken = [torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda") for n in (1 << 12, 1 << 14, 1 << 16, 1 << 18, 1 << 20, 1 << 21, 1 << 22) for _ in range(4)]
    canvas[out: late] = float(ops.SENTINEL)
    for t in (ent, rows_t, lp_t):
        t.zero_()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert plan.status() == 0
    got = [canvas[out: late], ent, rows_t, lp_t, plan.next_tokens(columns)]
    for a, b in zip(got[:4], want[:4]):
        assert torch.equal(a, b)
    assert np.array_equal(got[4], want[4])
    for t in taken:
        assert bool((t == 0x7f).all()), "the graph wrote into memory that is someone else's"
    del g
    plan.close()


def test_a_sequence_behind_the_last_column_is_refused():
    """One of no tokens too: its block of columns does not exist, so nothing would empty its cache column."""
    plan = NativePlan.create(512 * 64, 64, 20)
    cache = KV8Cache(4, 1, 64, 30)
    cache.views()["tail_block"].fill_(0)
    plan.add_kv8_fill(cache, 0, 64 * 64, 10)
    with pytest.raises(NativeError):
        plan.set_sequences([0, 1, 2], [10, 10, 0])
    plan.set_sequences([0, 1, -1], [10, 0, 0])                       # a block that exists may be empty
    plan.execute()
    assert plan.status() == 0
    assert cache.views()["tail_block"].flatten().tolist() == [0, -1, 0, 0]
    plan.close()
    plan = NativePlan.create(512 * 64, 64, 20)
    plan.set_sequences([0, 1, 2], [10, 10, 0])
    with pytest.raises(NativeError):
        plan.add_kv8_fill(cache, 0, 64 * 64, 10)                    # the sequences set before do not fit it
    plan.set_sequences([0, 1, 2], [9, 9, 0])
    plan.add_kv8_fill(cache, 0, 64 * 64, 9)
    plan.execute()
    assert plan.status() == 0
    assert cache.views()["tail_block"].flatten().tolist() == [0, 0, -1, 0]
    plan.close()


@pytest.mark.parametrize("stay", [False, True])
def test_positions_that_an_advancing_arg_max_moves_to_the_end(stay):
    """Without a limit a column runs out of the cache: it is idle then, its cache is left alone and the status says so; with one it stays
    at the last position. The other columns go on."""
    import torch
    h_q, h_kv, dim, max_seq = 2, 1, 64, 100
    positions = np.array([max_seq - 1, 5, -1, 62], dtype=np.int32)
    d = ops.Decoder(h_q, h_kv, dim, positions.size, max_seq, seed=21)
    d.history()
    d.cache.views()["tail_block"].copy_(torch.tensor([[1], [0], [-1], [0]], dtype=torch.int32))
    body = d.rng.normal(0, 1, (d.rq + 2 * d.rk, d.pitch)).astype(np.float16)
    d.canvas[: body.size] = torch.from_numpy(body.reshape(-1)).cuda()
    d.plan.add_argmax(0, d.rq, advance=True, max_seq=max_seq if stay else 0)
    d.plan.set_positions(positions)
    for step in range(3):
        before = ops.cache_arrays(d.cache)
        d.canvas[body.size:] = float(ops.SENTINEL)
        d.plan.execute_graph() if step else d.plan.execute()
        now = positions.copy()
        if step and stay:
            now[0] = max_seq - 1
        elif step:
            now[0] = -1                                                # what the kernels make of max_seq and beyond
        if stay or step == 0:
            assert d.plan.status() == 0
        else:
            with pytest.raises(NativeError, match="status 0x10:"):
                d.plan.status()
        d.check(now, body, ops.read(d.canvas, d.pitch)[body.shape[0]:, : d.columns], before, ops.cache_arrays(d.cache))
        positions[positions >= 0] += 1
    d.plan.close()


def fill_and_step(n, filled, dim, llama3=False, back=None):
    """The first `filled` of n tokens from a prompt, the others one by one, then one at position `back`; the cache's arrays."""
    import torch
    h_kv = 2
    rk = h_kv * dim
    data = np.random.default_rng(31).normal(0, 1, (2 * rk, 256)).astype(np.float16)
    cache = KV8Cache(1, h_kv, dim, 256)
    if filled:
        pitch = ops.pitch_of(filled)
        body = np.zeros((2 * rk, pitch), dtype=np.float16)
        body[:, :filled] = data[:, :filled]
        plan, _ = ops.make_plan(body, 0, filled)
        plan.add_kv8_fill(cache, 0, rk * pitch, filled, theta=ops.THETA, llama3=llama3)
        plan.set_sequences([0], [filled])
        plan.execute()
        assert plan.status() == 0
        plan.close()
    body = np.ones((3 * rk, 64), dtype=np.float16)
    plan, canvas = ops.make_plan(body, rk, 1)
    plan.add_kv8_attn(cache, 0, rk * 64, 2 * rk * 64, 3 * rk * 64, h_kv, theta=ops.THETA, llama3=llama3)
    steps = [(t, t) for t in range(filled, n)] + ([] if back is None else [(back, 255)])
    for t, token in steps:
        canvas.view(-1, 64)[rk: 3 * rk, 0] = torch.from_numpy(data[:, token].copy()).cuda()
        plan.set_positions([t])
        plan.execute()
    assert plan.status() == 0
    out = ops.read(canvas, 64)[3 * rk:, 0].copy()
    plan.close()
    return ops.cache_arrays(cache), out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("llama3", [False, True])
def test_a_prompt_and_tokens_leave_the_same_bits(dim, llama3):
    n = 150
    want, out = fill_and_step(n, 0, dim, llama3)
    rest = n % 64
    for filled in (149, 128, 100, 64, 63, 1):
        got, o = fill_and_step(n, filled, dim, llama3)
        assert np.array_equal(got["codes"][:, :, :2], want["codes"][:, :, :2]) and np.array_equal(got["scales"][:, :, :2], want["scales"][:, :, :2])
        assert np.array_equal(got["k_tail"][:, :, :rest], want["k_tail"][:, :, :rest]) and np.array_equal(got["v_tail"][..., :rest], want["v_tail"][..., :rest])
        assert np.array_equal(got["tail_block"], want["tail_block"]) and np.array_equal(o, out)
    # and they are the keys at their positions
    k = np.random.default_rng(31).normal(0, 1, (4 * dim, 256)).astype(np.float16)[:dim, 128:n].astype(np.float64).T
    k = D.rotated(k, np.arange(128, n), ops.THETA, llama3)
    assert np.all(np.abs(want["k_tail"][0, 0, :rest] - k) <= D.HALF16 * np.abs(k) + 2.0 ** -22 * np.abs(k).max() + D.TINY16)


@pytest.mark.parametrize("dim", [64, 128])
def test_going_back_into_a_block_that_has_just_been_completed(dim):
    """Its FP16 rows are still there until a token of another block comes; after that, or where a prompt filled it, it starts from its 8 bits."""
    back = 40
    kept, _ = fill_and_step(128, 0, dim)
    rows, out_rows = fill_and_step(128, 0, dim, back=64 + back)
    assert np.array_equal(rows["k_tail"][:, :, :back], kept["k_tail"][:, :, :back]) and np.array_equal(rows["v_tail"][..., :back], kept["v_tail"][..., :back])
    filled, out_filled = fill_and_step(128, 128, dim, back=64 + back)
    for h in range(2):
        k, v = ops.block_values(kept, 0, h, 1, dim)
        assert np.array_equal(filled["k_tail"][0, h, :back], k[:back].astype(np.float32).astype(np.float16))
        assert np.array_equal(filled["v_tail"][0, h, :, :back].T, v[:back].astype(np.float32).astype(np.float16))
    assert np.array_equal(filled["k_tail"][:, :, back], rows["k_tail"][:, :, back]) and (rows["tail_block"] == 1).all() and (filled["tail_block"] == 1).all()
    later, out_later = fill_and_step(129, 0, dim, back=64 + back)
    assert np.array_equal(later["k_tail"][:, :, :back], filled["k_tail"][:, :, :back]) and np.array_equal(later["v_tail"][..., :back], filled["v_tail"][..., :back])
    assert np.array_equal(out_later, out_filled) and np.isfinite(out_rows).all()
