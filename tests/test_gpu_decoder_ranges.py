"""The decoder operators at the ends of their numbers' ranges: weights far below the largest, scores of some tens, queries and keys whose
rotation leaves FP16, values that are not finite. Against the 64-bit oracle, whose bounds follow from the kernels' roundings."""
import numpy as np
import pytest

import test_gpu_decoder_ops as ops
from oracle import decoder as D

pytestmark = pytest.mark.gpu


# ---- weights far below the largest ---------------------------------------------------------------------------------------------------
def blocks_of_8_bits(x):
    """x [..., 64, dim] on the GPU -> codes and scales of the cache's format."""
    import torch
    scale = x.abs().amax(dim=(-2, -1)).clamp_min(2.0 ** -24) / 448.0
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


@pytest.mark.parametrize("h_q,h_kv,dim,columns", [(8, 8, 64, 64), (16, 4, 128, 64), (16, 1, 64, 192), (16, 1, 128, 192)])
def test_a_loud_block_leaves_the_weights_of_the_others(h_q, h_kv, dim, columns):
    """Every fifth block holds one value of 6e4 and a token that leads by 6 to 10 nats, so that the others' weights, times their values'
    scale, are as small as 2^-28 of that block's; a warp's share is some 17 blocks, which hold several of both kinds. Magnitudes of the
    other blocks differ by up to 10^4."""
    import torch
    blocks = 30000 // (columns * h_kv)
    pos = blocks * 64 + 20
    d = ops.Decoder(h_q, h_kv, dim, columns, pos + 5, seed=41)
    g = torch.Generator(device="cuda").manual_seed(42)
    group = h_q // h_kv
    # the same query for all heads of a column, and keys of two kinds: along it (rotated), and nothing
    body = np.zeros((d.rq + 2 * d.rk, d.pitch), dtype=np.float16)
    one = d.rng.normal(0, 1, (dim, columns)).astype(np.float16)
    body[: d.rq, :columns] = np.tile(one, (h_q, 1))
    body[d.rq + d.rk:, :columns] = d.rng.normal(0.01, 0.002, (d.rk, columns)).astype(np.float16)
    q = D.rotated(one.astype(np.float64).T, np.full(columns, pos), ops.THETA)
    lead = 6.0 + 4.0 * np.arange(columns) / columns
    unit = torch.from_numpy(q * (lead * np.sqrt(dim) / (q * q).sum(axis=1))[:, None]).cuda().float()
    v = d.cache.views()
    for c in range(columns):
        k = torch.zeros(h_kv, blocks + 1, 64, dim, device="cuda")
        size = 10.0 ** -(torch.arange(blocks + 1, device="cuda") % 5).float()
        x = (1.0 + 0.1 * torch.randn(h_kv, blocks + 1, 64, dim, generator=g, device="cuda")) * size[:, None, None]
        k[:, ::5, 9] = unit[c]
        x[:, ::5, 30, 7] = 6e4
        kc, ks = blocks_of_8_bits(k)
        xc, xs = blocks_of_8_bits(x)
        v["codes"].view(torch.uint8)[c, :, :, 0] = kc.view(torch.uint8).unflatten(-1, (dim // 64, 64)).transpose(-3, -2).flatten(-3)
        v["codes"].view(torch.uint8)[c, :, :, 1] = xc.view(torch.uint8).transpose(-2, -1).flatten(-2)
        v["scales"][c, :, :, 0], v["scales"][c, :, :, 1] = ks, xs
    v["k_tail"].zero_()
    v["v_tail"].fill_(0.01)
    out = d.step(np.full(columns, pos), check=False, body=body)
    a = ops.cache_arrays(d.cache)
    for c, h in [(0, 0), (columns // 3, h_kv // 2), (columns // 2 + 1, 0), (columns - 1, h_kv - 1)]:
        parts = [ops.block_values(a, c, h, i, dim) for i in range(blocks)]
        K = np.concatenate([i[0] for i in parts] + [a["k_tail"][c, h, :21].astype(np.float64)])
        V = np.concatenate([i[1] for i in parts] + [a["v_tail"][c, h, :, :21].astype(np.float64).T])
        want, bound = D.attend(np.repeat(q[c: c + 1], group, 0), K, V, np.ones((group, pos + 1), dtype=bool), 2.0 ** -21 + dim * 2.0 ** -23, least_weight=2.0 ** -39)
        ops.within(out[h * group * dim: (h + 1) * group * dim, c].reshape(group, dim), want, bound, f"column {c} head {h}")
    d.plan.close()


@pytest.mark.parametrize("h_q,dim", [(4, 64), (16, 128)])
def test_blocks_of_a_cleared_cache_are_zeros(h_q, dim):
    """A code times its scale, 0 times 0: tokens that nobody appended have weights like others, and values of nothing."""
    d = ops.Decoder(h_q, 1, dim, 3, 300, seed=9)
    d.step([130, 64, 299])
    d.step([131, 65, 5])
    d.plan.close()


@pytest.mark.parametrize("h_q,dim", [(4, 64), (16, 128)])
def test_blocks_of_a_cleared_cache_at_the_edges_of_a_window(h_q, dim):
    d = ops.Decoder(h_q, 1, dim, 3, 300, 60, 100, seed=10)
    d.step([216, 130, 299])
    d.step([217, 131, 110])
    d.plan.close()


@pytest.mark.parametrize("dim", [64, 128])
def test_one_key_far_above_the_others(dim):
    """A first key that leads by 6 to 17 nats and whose value is nothing: the output is made of weights as small as 2^-24 of the largest."""
    leads = [6.0, 9.0, 11.0, 13.0, 15.0, 17.0]
    heads, seq = len(leads), 1500
    rng = np.random.default_rng(dim)
    pitch, r = ops.pitch_of(seq), heads * dim
    body = np.zeros((3 * r, pitch), dtype=np.float16)
    for h, lead in enumerate(leads):          # only the slowest pair, which a large base leaves where it is
        body[h * dim + dim // 2 - 1] = np.sqrt(dim)
        body[r + h * dim + dim // 2 - 1, 0] = lead
    body[2 * r:] = rng.normal(1, 0.1, (r, pitch)).astype(np.float16)
    body[2 * r:, 0] = 0
    plan, canvas = ops.make_plan(body, r, seq)
    plan.add_window_attn(0, r * pitch, 2 * r * pitch, 3 * r * pitch, heads, heads, dim, seq, theta=1e30)
    plan.execute()
    assert plan.status() == 0
    x = body[:, :seq].astype(np.float64)
    want, bound = D.window_attention(x[:r], x[r: 2 * r], x[2 * r:], heads, heads, seq, seq, 0, 0, 1e30)
    ops.within(ops.read(canvas, pitch)[3 * r:, :seq], want, bound, "window attention")
    plan.close()


# ---- scores of some tens --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,window,size", [(64, 0, 3.0), (128, 0, 3.0), (64, 200, 4.0), (128, 77, 2.5)])
def test_scores_of_some_tens(dim, window, size):
    """Maxima that keep growing: queries and keys of `size`, scores of about its square."""
    h_q, h_kv, seq, columns = 4, 2, 700, 1400
    rng = np.random.default_rng(dim + window)
    pitch, rq, rk = ops.pitch_of(columns), h_q * dim, h_kv * dim
    body = rng.normal(0, 1, (rq + 2 * rk, pitch)).astype(np.float16)
    body[: rq + rk] *= np.float16(size)
    plan, canvas = ops.make_plan(body, rq, columns)
    plan.add_window_attn(0, rq * pitch, (rq + rk) * pitch, (rq + 2 * rk) * pitch, h_q, h_kv, dim, seq, window=window, sinks=3, theta=ops.THETA)
    plan.execute()
    assert plan.status() == 0
    x = body[:, :columns].astype(np.float64)
    want, bound = D.window_attention(x[:rq], x[rq: rq + rk], x[rq + rk:], h_q, h_kv, seq, columns, window, 3, ops.THETA)
    ops.within(ops.read(canvas, pitch)[rq + 2 * rk:, :columns], want, bound, "window attention")
    plan.close()


# ---- rotations that leave FP16 --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("loud", ["queries", "keys"])
def test_window_attention_with_rotations_beyond_fp16(dim, loud):
    """A pair of 6e4 and 6e4 is as long as 84852, which is no FP16 number; the scores are ordinary."""
    seq, columns = 150, 290
    rng = np.random.default_rng(dim)
    pitch = ops.pitch_of(columns)
    body = rng.normal(0, 1, (3 * dim, pitch)).astype(np.float16)
    big, small = (0, dim) if loud == "queries" else (dim, 0)
    body[big: big + dim] = 0
    for p in (0, 5, dim // 2 - 1):
        body[big + p], body[big + p + dim // 2] = 60000, rng.choice([-60000, 60000], pitch)
    body[small: small + dim] *= np.float16(2.0 ** -10)
    plan, canvas = ops.make_plan(body, dim, columns)
    plan.add_window_attn(0, dim * pitch, 2 * dim * pitch, 3 * dim * pitch, 1, 1, dim, seq, theta=ops.THETA)
    plan.execute()
    assert plan.status() == 0
    x = body[:, :columns].astype(np.float64)
    want, bound = D.window_attention(x[:dim], x[dim: 2 * dim], x[2 * dim:], 1, 1, seq, columns, 0, 0, ops.THETA)
    assert np.isfinite(want).all() and np.median(bound) < 0.2, "the bound says something"
    ops.within(ops.read(canvas, pitch)[3 * dim:, :columns], want, bound, "window attention")
    plan.close()


@pytest.mark.parametrize("h_q,dim", [(4, 64), (12, 64), (2, 128), (16, 128)])
def test_kv8_attention_with_queries_beyond_fp16(h_q, dim):
    """As above for the queries of single tokens."""
    positions = np.array([1, 5, 63, 64, 130, 200], dtype=np.int32)
    d = ops.Decoder(h_q, 1, dim, positions.size, 256, seed=dim)
    d.history()
    v = d.cache.views()
    v["scales"][..., 0] *= 2.0 ** -12
    v["k_tail"].mul_(2.0 ** -10)
    body = d.rng.normal(0, 1, (d.rq + 2 * dim, d.pitch)).astype(np.float16)
    body[: d.rq] = 0
    for h in range(h_q):
        body[h * dim + 3], body[h * dim + 3 + dim // 2] = 60000, d.rng.choice([-60000, 60000], d.pitch)
    body[d.rq: d.rq + dim] *= np.float16(2.0 ** -10)
    d.step(positions, body=body)
    d.plan.close()


@pytest.mark.parametrize("dim", [64, 128])
def test_cached_keys_beyond_fp16_are_held_as_the_largest_number(dim):
    """Finite keys stay finite, from a prompt and token by token; an infinity stays one in the open block."""
    import torch
    n, h_kv = 70, 2
    rk, pitch = h_kv * dim, 128
    rng = np.random.default_rng(dim)
    body = rng.normal(0, 1, (2 * rk, pitch)).astype(np.float16)
    body[4, :], body[4 + dim // 2, :] = 60000, rng.choice([-60000, 60000], pitch)
    body[rk - 1, 66] = np.inf
    cache = ops.KV8Cache(1, h_kv, dim, 128)
    plan, _ = ops.make_plan(body, 0, n)
    plan.add_kv8_fill(cache, 0, rk * pitch, n, theta=ops.THETA)
    plan.set_sequences([0], [n])
    plan.execute()
    assert plan.status() == 0
    plan.close()
    a = ops.cache_arrays(cache)
    k = D.rotated(body[:dim, :n].astype(np.float64).T, np.arange(n), ops.THETA)
    assert np.abs(k).max() > 80000
    held = np.clip(k, -65504, 65504)
    row = a["k_tail"][0, 0, :6].astype(np.float64)
    assert np.all(np.abs(row - held[64:]) <= D.HALF16 * np.abs(held[64:]) + 2.0 ** -22 * np.abs(k).max() + D.TINY16)
    assert np.isinf(a["k_tail"][0, 1, 2, dim - 1]), "an infinity"
    got = ops.block_values(a, 0, 0, 0, dim)[0]
    assert abs(a["scales"][0, 0, 0, 0] / (65504 / 448) - 1) <= 2.0 ** -23
    scale = 65504 / 448
    assert np.all(np.abs(got - held[:64]) <= (D.e4m3_half_step(np.abs(held[:64]) / scale * (1 + 2 * D.HALF16)) * scale + D.HALF16 * np.abs(held[:64]) * 1.01 + 2.0 ** -22 * np.abs(k).max()) * 1.001)
    # the same tokens one by one
    one = ops.Decoder(h_kv, h_kv, dim, 1, 128)
    for t in range(n):
        x = np.zeros((3 * rk, one.pitch), dtype=np.float16)
        x[rk:, 0] = body[:, t]
        one.step([t], tag=False, check=False, body=x)
    for part, b in ops.cache_arrays(one.cache).items():
        if part != "tail_block":
            assert np.array_equal(b[..., :6, :] if part == "k_tail" else b[..., :6] if part == "v_tail" else b[:, :, :1], a[part][..., :6, :] if part == "k_tail" else a[part][..., :6] if part == "v_tail" else a[part][:, :, :1], equal_nan=part != "codes"), part
    one.plan.close()


# ---- values that are not finite ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,columns,seq,window,sinks", [(64, 1000, 500, 0, 0), (128, 1000, 500, 0, 0), (64, 900, 900, 150, 70), (128, 333, 111, 0, 0), (64, 70, 70, 0, 0)])
def test_values_that_are_not_finite_reach_the_columns_that_see_them(dim, columns, seq, window, sinks):
    """One of a kind in some tiles, a whole tile of them, the first and last columns of tiles, hidden ones between seen ones."""
    h_q, h_kv = 4, 2
    rng = np.random.default_rng(columns + dim)
    pitch, rq, rk = ops.pitch_of(columns), h_q * dim, h_kv * dim
    body = rng.normal(0, 1, (rq + 2 * rk, pitch)).astype(np.float16)
    v = body[rq + rk:]
    for c in (0, 7, 8, 63, 64, 127, 300, 447, 448, 499, 500, 512, 640, 899):
        if c < columns:
            v[rng.integers(0, rk), c] = rng.choice([np.inf, -np.inf, np.nan])
    v[rk - 1, 320: 384] = np.nan
    v[3, columns - 1], v[3, columns - 2] = np.inf, -np.inf
    v[:, columns:] = np.nan
    plan, canvas = ops.make_plan(body, rq, columns)
    plan.add_window_attn(0, rq * pitch, (rq + rk) * pitch, (rq + 2 * rk) * pitch, h_q, h_kv, dim, seq, window=window, sinks=sinks, theta=ops.THETA)
    plan.execute()
    assert plan.status() == 0
    x = body[:, :columns].astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, bound = D.window_attention(x[:rq], x[rq: rq + rk], x[rq + rk:], h_q, h_kv, seq, columns, window, sinks, ops.THETA)
    assert not np.isfinite(want).all()
    ops.within(ops.read(canvas, pitch)[rq + 2 * rk:, :columns], want, bound, "window attention")
    plan.close()


@pytest.mark.parametrize("dim", [64, 128])
def test_odd_keys_and_values_from_a_prompt_and_token_by_token(dim):
    """Infinities, NaN and numbers at the end of FP16 in complete blocks and in the open one leave the same codes, scales and rows (the code
    of a NaN may have either sign)."""
    import torch
    h_kv, n, pitch = 3, 200, 256
    rk = h_kv * dim
    rng = np.random.default_rng(dim)
    body = rng.normal(0, 1, (2 * rk, pitch)).astype(np.float16)
    for x in (np.nan, np.inf, -np.inf, 65504, -60000):
        for _ in range(6):
            body[rng.integers(0, 2 * rk), rng.integers(0, n)] = x
    prompt = ops.KV8Cache(1, h_kv, dim, 256)
    plan, _ = ops.make_plan(body, 0, n)
    plan.add_kv8_fill(prompt, 0, rk * pitch, n, theta=ops.THETA)
    plan.set_sequences([0], [n])
    plan.execute()
    assert plan.status() == 0
    plan.close()
    one = ops.Decoder(h_kv, h_kv, dim, 1, 256)
    for t in range(n):
        x = np.zeros((3 * rk, one.pitch), dtype=np.float16)
        x[rk:, 0] = body[:, t]
        one.step([t], tag=False, check=False, body=x)
    a, b = ops.cache_arrays(prompt), ops.cache_arrays(one.cache)
    r, whole = n % 64, n // 64
    nan = (a["codes"][:, :, :whole] & 127) == 127
    assert nan.any() and np.array_equal(nan, (b["codes"][:, :, :whole] & 127) == 127)
    assert np.array_equal(a["codes"][:, :, :whole][~nan], b["codes"][:, :, :whole][~nan]) and np.array_equal(a["scales"][:, :, :whole], b["scales"][:, :, :whole])
    assert np.array_equal(a["k_tail"][:, :, :r], b["k_tail"][:, :, :r], equal_nan=True) and np.array_equal(a["v_tail"][..., :r], b["v_tail"][..., :r], equal_nan=True)
    one.plan.close()
