"""GPU parity of the decoder operators (prompt attention with a window and sinks, the 8-bit key / value cache, answer probabilities),
called through the C ABI, against the 64-bit oracle (oracle/decoder.py). Tolerances are the oracle's error bounds: they follow from the
inputs and the kernels' roundings."""
import numpy as np
import pytest

from oracle import decoder as D
from snntome_b200.native import KV8Cache, NativeError, NativePlan

pytestmark = pytest.mark.gpu
THETA = 10000.0
SENTINEL = np.float16(-77.0)


def make_plan(body, rows_out, columns):
    """A plan whose canvas holds `body` [rows][pitch] (FP16) and behind it `rows_out` rows of a sentinel."""
    import torch
    rows, pitch = body.shape
    plan = NativePlan.create((rows + rows_out) * pitch, pitch, columns)
    canvas = plan.canvas_tensor()
    canvas[: rows * pitch] = torch.from_numpy(body.reshape(-1)).cuda()
    canvas[rows * pitch:] = float(SENTINEL)
    return plan, canvas


def pitch_of(columns):
    return (columns + 63) // 64 * 64


def read(canvas, pitch):
    return canvas.cpu().numpy().reshape(-1, pitch)


def within(got, want, bound, what):
    """NaN and infinite values must be in the same places; the rest within the bound."""
    got = np.asarray(got, dtype=np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    off = np.abs(got[fine] - want[fine]) - np.broadcast_to(bound, want.shape)[fine]
    assert off.size == 0 or off.max() <= 0, f"{what}: {off.max()} beyond the bound {np.broadcast_to(bound, want.shape)[fine][int(off.argmax())]}"


# ---- prompt attention -----------------------------------------------------------------------------------------------------------
WINDOW_CASES = [(4, 2, 64, 1, 5, 0, 0), (2, 1, 64, 100, 100, 0, 0), (8, 2, 64, 37, 200, 0, 0), (4, 4, 128, 130, 390, 16, 3), (3, 1, 64, 300, 300, 64, 0),
                (16, 2, 64, 513, 513, 100, 130), (2, 2, 128, 64, 64, 1, 0), (5, 1, 64, 1000, 700, 128, 4), (2, 1, 64, 700, 700, 200, 200), (1, 1, 128, 1100, 1100, 0, 0),
                (2, 1, 64, 640, 1280, 1000, 7), (1, 1, 64, 4096, 1, 5, 5), (2, 2, 64, 129, 516, 129, 1), (1, 1, 128, 900, 900, 1, 257)]


@pytest.mark.parametrize("h_q,h_kv,dim,seq,columns,window,sinks", WINDOW_CASES)
def test_window_attention(h_q, h_kv, dim, seq, columns, window, sinks):
    rng = np.random.default_rng(seq * 31 + window)
    pitch, rq, rk = pitch_of(columns), h_q * dim, h_kv * dim
    body = rng.normal(0, 1, (rq + 2 * rk, pitch)).astype(np.float16)
    body[:, columns:] = np.nan                                  # what lies behind the last column must not matter
    plan, canvas = make_plan(body, rq + 1, columns)
    o = (rq + 2 * rk) * pitch
    plan.add_window_attn(0, rq * pitch, (rq + rk) * pitch, o, h_q, h_kv, dim, seq, window=window, sinks=sinks, theta=THETA)
    plan.execute()
    assert plan.status() == 0
    got = read(canvas, pitch)
    x = body[:, :columns].astype(np.float64)
    want, bound = D.window_attention(x[:rq], x[rq: rq + rk], x[rq + rk:], h_q, h_kv, seq, columns, window, sinks, THETA)
    within(got[rq + 2 * rk: 2 * rq + 2 * rk, :columns], want, bound, "window attention")
    assert np.array_equal(got[: rq + 2 * rk].view(np.uint16), body.view(np.uint16)), "q, k and v stay as they were"
    assert (got[rq + 2 * rk:, columns:] == SENTINEL).all() and (got[-1] == SENTINEL).all(), "nothing else is written"
    first = got.copy()
    plan.execute_graph()
    plan.execute_graph()
    assert np.array_equal(read(canvas, pitch).view(np.uint16), first.view(np.uint16)), "every run gives the same bits"
    plan.close()


def test_window_attention_hidden_columns_do_not_count():
    h_q, h_kv, dim, seq, columns, window, sinks = 2, 1, 64, 450, 900, 40, 3
    rng = np.random.default_rng(9)
    pitch, rq, rk = pitch_of(columns), h_q * dim, h_kv * dim
    body = rng.normal(0, 1, (rq + 2 * rk, pitch)).astype(np.float16)
    body[rq + rk + 5, 100] = np.nan                             # a value: seen by columns 100 .. 139 of the first sequence
    body[rq + rk + 9, 101] = np.inf
    body[rq + rk + 9, 120] = -np.inf                            # meets the one above: NaN for the columns that see both
    body[rq + 3, 300] = np.nan                                  # a key
    body[rq + rk + 7, 451] = np.inf                             # a sink of the second sequence
    body[rq + 1, 899] = np.inf
    body[5, 200] = np.nan                                       # a query: its own column only
    plan, canvas = make_plan(body, rq, columns)
    plan.add_window_attn(0, rq * pitch, (rq + rk) * pitch, (rq + 2 * rk) * pitch, h_q, h_kv, dim, seq, window=window, sinks=sinks, theta=THETA, llama3=True)
    plan.execute()
    assert plan.status() == 0
    x = body[:, :columns].astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, bound = D.window_attention(x[:rq], x[rq: rq + rk], x[rq + rk:], h_q, h_kv, seq, columns, window, sinks, THETA, True)
    assert np.isfinite(want[5, 99]) and np.isnan(want[5, 139]) and np.isfinite(want[5, 140]) and want[9, 110] == np.inf and np.isnan(want[9, 130]) and want[7, 890] == np.inf
    within(read(canvas, pitch)[rq + 2 * rk:, :columns], want, bound, "window attention")
    plan.close()


@pytest.mark.parametrize("dim,window", [(64, 0), (128, 0), (64, 300), (128, 300)])
def test_window_attention_with_every_multiprocessor_busy(dim, window):
    """Long rows on more CTAs than fit at once, whose warps drift apart: many runs, one result, and the right one."""
    import torch
    h_q, h_kv, seq, columns = 32, 8, 1000, 3000
    rng = np.random.default_rng(dim + window)
    pitch, rq, rk = pitch_of(columns), h_q * dim, h_kv * dim
    body = rng.normal(0, 1, (rq + 2 * rk, pitch)).astype(np.float16)
    plan, canvas = make_plan(body, rq, columns)
    o = (rq + 2 * rk) * pitch
    plan.add_window_attn(0, rq * pitch, (rq + rk) * pitch, o, h_q, h_kv, dim, seq, window=window, sinks=4, theta=THETA)
    plan.execute()
    first = canvas.clone()
    for i in range(30):
        canvas[o:] = float(SENTINEL)
        plan.execute() if i % 2 else plan.execute_graph()
        assert torch.equal(canvas.view(torch.int16), first.view(torch.int16)), "every run gives the same bits"
    assert plan.status() == 0
    got = read(canvas, pitch)
    x = body[:, :columns].astype(np.float64)
    for h in (0, 13, 31):
        k = h // (h_q // h_kv)
        want, bound = D.window_attention(x[h * dim: (h + 1) * dim], x[rq + k * dim: rq + (k + 1) * dim], x[rq + rk + k * dim: rq + rk + (k + 1) * dim], 1, 1, seq, columns, window, 4, THETA)
        within(got[rq + 2 * rk + h * dim: rq + 2 * rk + (h + 1) * dim, :columns], want, bound, f"window attention, head {h}")
    plan.close()


# ---- the cache ---------------------------------------------------------------------------------------------------------------------
def cache_arrays(cache):
    import torch
    v = cache.views()
    return dict(codes=v["codes"].view(torch.uint8).cpu().numpy(), scales=v["scales"].cpu().numpy(), k_tail=v["k_tail"].cpu().numpy(),
                v_tail=v["v_tail"].cpu().numpy(), tail_block=v["tail_block"].cpu().numpy())


def block_values(a, col, h, b, dim):
    """Keys and values [64, dim] of an 8-bit block, in 64 bits."""
    t = D.e4m3_values()
    k = t[a["codes"][col, h, b, 0]].reshape(dim // 64, 64, 64).transpose(1, 0, 2).reshape(64, dim) * np.float64(a["scales"][col, h, b, 0])
    v = t[a["codes"][col, h, b, 1]].reshape(dim, 64).T * np.float64(a["scales"][col, h, b, 1])
    return k, v


def check_block(a, col, h, b, k, v, what):
    """An 8-bit block against the FP16 keys and values [64, dim] that it stands for (each off by up to half a step of e4m3)."""
    dim = k.shape[1]
    gk, gv = block_values(a, col, h, b, dim)
    for got, x, i in ((gk, k, 0), (gv, v, 1)):
        scale = np.float64(a["scales"][col, h, b, i])
        assert abs(scale / D.block_scale(x) - 1) <= 2.0 ** -23, f"{what}: scale"
        x = np.clip(x, -65504, 65504)
        fine = np.isfinite(x)
        assert np.array_equal(np.isnan(got), ~fine), f"{what}: NaN"
        assert np.all(np.abs(got - x)[fine] <= (D.e4m3_half_step(x / scale) * scale * D.CODE_SLACK)[fine]), f"{what}: codes"


@pytest.mark.parametrize("h_kv,dim,seq,frames,columns,max_seq", [(2, 64, 200, 3, 5, 256), (1, 128, 77, 4, 4, 77), (3, 64, 64, 2, 2, 64), (1, 64, 1, 3, 3, 5), (2, 128, 515, 1, 2, 1000)])
def test_fill(h_kv, dim, seq, frames, columns, max_seq):
    import torch
    rng = np.random.default_rng(dim + seq)
    cols, rk = frames * seq, h_kv * dim
    pitch = pitch_of(cols)
    body = (rng.normal(0, 1, (2 * rk, pitch)) * np.exp(rng.normal(0, 1, (2 * rk, 1)))).astype(np.float16)
    body[: rk, : 3] = 0
    slots = rng.permutation(columns)[:frames].astype(np.int32)
    lengths = np.array([seq, rng.integers(0, seq + 1), 0, seq // 2][:frames], dtype=np.int32)
    if frames == 4:
        slots[1] = -1
    cache = KV8Cache(columns, h_kv, dim, max_seq)
    cache.storage.copy_(torch.from_numpy(rng.integers(0, 120, cache.storage.numel(), dtype=np.uint8)))
    before = cache_arrays(cache)
    plan, canvas = make_plan(body, 0, cols)
    plan.add_kv8_fill(cache, 0, rk * pitch, seq, theta=THETA)
    plan.set_sequences(slots, lengths)
    plan.execute()
    assert plan.status() == 0
    a = cache_arrays(cache)
    touched = {k: np.zeros(v.shape, dtype=bool) for k, v in a.items()}
    for f in range(frames):
        if slots[f] < 0:
            continue
        n, c = int(lengths[f]), int(slots[f])
        at = slice(f * seq, f * seq + n)
        for h in range(h_kv):
            touched["tail_block"][c, h] = True
            assert a["tail_block"][c, h] == (n // 64 if n % 64 else -1)
            if n == 0:
                continue
            k = D.rotated(body[h * dim: (h + 1) * dim, at].astype(np.float64).T, np.arange(n), THETA)
            v = body[rk + h * dim: rk + (h + 1) * dim, at].astype(np.float64).T
            r = n % 64
            if r:
                touched["k_tail"][c, h, :r] = touched["v_tail"][c, h, :, :r] = True
                # half a step of FP16 and the 32-bit rotation
                assert np.all(np.abs(a["k_tail"][c, h, :r] - k[-r:]) <= D.HALF16 * np.abs(k[-r:]) + 2.0 ** -22 * np.abs(k).max() + D.TINY16)
                assert np.array_equal(a["v_tail"][c, h, :, :r].T, v[-r:])
            for b in range(n // 64):
                touched["codes"][c, h, b] = touched["scales"][c, h, b] = True
                kb, vb = k[b * 64: b * 64 + 64], v[b * 64: b * 64 + 64]
                gk, gv = block_values(a, c, h, b, dim)
                ks = np.float64(a["scales"][c, h, b, 0])
                assert abs(ks / D.block_scale(kb) - 1) <= D.HALF16 * 1.01
                # the key is rounded to FP16, then to e4m3
                step = D.e4m3_half_step(np.abs(kb / ks) * (1 + 2 * D.HALF16)) * ks + D.HALF16 * np.abs(kb) * 1.01 + 2.0 ** -22 * np.abs(k).max() + D.TINY16
                assert np.all(np.abs(gk - kb) <= step * 1.001)
                vs = np.float64(a["scales"][c, h, b, 1])
                assert abs(vs / D.block_scale(vb) - 1) <= 2.0 ** -23
                assert np.all(np.abs(gv - vb) <= D.e4m3_half_step(vb / vs) * vs * D.CODE_SLACK)
    for part in a:
        same = a[part].view(np.uint8).reshape(*a[part].shape, -1) == before[part].view(np.uint8).reshape(*a[part].shape, -1)
        assert same[~touched[part]].all(), f"{part}: something else was written"
    plan.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq,max_seq", [(133, 133), (141, 133), (203, 135), (134, 1000)])
def test_fill_from_any_column(dim, seq, max_seq):
    """Sequences that start on odd columns, and plans whose sequences are longer than the cache, leave the bits that aligned ones leave."""
    import torch
    h_kv, lengths = 3, np.array([133, 64, 128, 1, 70, 131, 0, 40, 129], dtype=np.int32)
    rng = np.random.default_rng(seq + dim)
    rk, frames = h_kv * dim, len(lengths)
    data = rng.normal(0, 1, (2 * rk, frames, 133)).astype(np.float16)
    got = []
    for s in (192, seq):
        pitch = pitch_of(frames * s)
        body = np.full((2 * rk, pitch), np.nan, dtype=np.float16)          # what lies between the sequences must not matter
        for f, n in enumerate(lengths):
            body[:, f * s: f * s + n] = data[:, f, :n]
        cache = KV8Cache(frames, h_kv, dim, max_seq)
        cache.storage.fill_(77)
        plan, canvas = make_plan(body, 0, frames * s)
        plan.add_kv8_fill(cache, 0, rk * pitch, s, theta=THETA)
        plan.set_sequences(np.arange(frames, dtype=np.int32)[::-1].copy(), lengths)
        plan.execute()
        assert plan.status() == 0
        got.append(cache.storage.clone())
        plan.close()
    assert torch.equal(got[0], got[1])


class Decoder:
    """A plan with one kv8_attn over a cache that random tokens fill step by step, and the oracle's view of it."""

    def __init__(self, h_q, h_kv, dim, columns, max_seq, window=0, sinks=0, seed=0, cache=None):
        self.h_q, self.h_kv, self.dim, self.columns, self.window, self.sinks = h_q, h_kv, dim, columns, window, sinks
        self.pitch, self.rq, self.rk = pitch_of(columns), h_q * dim, h_kv * dim
        self.rng = np.random.default_rng(seed)
        self.cache = cache or KV8Cache(columns, h_kv, dim, max_seq)
        self.plan, self.canvas = make_plan(np.zeros((self.rq + 2 * self.rk, self.pitch), dtype=np.float16), self.rq, columns)
        p = self.pitch
        self.plan.add_kv8_attn(self.cache, 0, self.rq * p, (self.rq + self.rk) * p, (self.rq + 2 * self.rk) * p, h_q, window=window, sinks=sinks, theta=THETA)

    def history(self, loud=4.0):
        """Random earlier positions in every column: 8-bit blocks and open blocks."""
        import torch
        v = self.cache.views()
        codes = self.rng.integers(0, 256, tuple(v["codes"].shape), dtype=np.uint8)
        codes[(codes & 127) == 127] = 0
        v["codes"].view(torch.uint8).copy_(torch.from_numpy(codes))
        v["scales"].copy_(torch.from_numpy(self.rng.uniform(0.001, 0.01, tuple(v["scales"].shape)).astype(np.float32)))
        v["k_tail"].copy_(torch.from_numpy(self.rng.normal(0, 1, tuple(v["k_tail"].shape)).astype(np.float16)))
        v["v_tail"].copy_(torch.from_numpy(self.rng.normal(0, loud, tuple(v["v_tail"].shape)).astype(np.float16)))

    def step(self, positions, graph=False, tag=True, check=True, body=None):
        import torch
        positions = np.asarray(positions, dtype=np.int32)
        if body is None:
            body = self.rng.normal(0, 1, (self.rq + 2 * self.rk, self.pitch)).astype(np.float16)
        self.body = body
        self.canvas[: body.size] = torch.from_numpy(body.reshape(-1)).cuda()
        self.canvas[body.size:] = float(SENTINEL)
        if tag:                                   # the open block is that of the position before
            t = np.where(positions > 0, (positions - 1) // 64, -1).astype(np.int32)
            self.cache.views()["tail_block"].copy_(torch.from_numpy(np.repeat(t[:, None], self.h_kv, 1)))
        before = cache_arrays(self.cache)
        self.plan.set_positions(positions)
        (self.plan.execute_graph if graph else self.plan.execute)()
        assert self.plan.status() == 0
        got = read(self.canvas, self.pitch)
        assert np.array_equal(got[: body.shape[0]].view(np.uint16), body.view(np.uint16)), "q, k and v stay as they were"
        out = got[body.shape[0]:]
        assert (out[:, self.columns:] == SENTINEL).all(), "columns behind the plan's last one"
        if check:
            self.check(positions, body, out, before, cache_arrays(self.cache))
        return out[:, : self.columns]

    def check(self, positions, body, out, before, a):
        dim, g = self.dim, self.h_q // self.h_kv
        x = body.astype(np.float64)
        for c, p in enumerate(positions):
            p = int(p)
            if p < 0:
                assert not out[:, c].any(), "an idle column gets zeros"
                for part in a:
                    assert np.array_equal(a[part][c].view(np.uint8), before[part][c].view(np.uint8)), f"idle column, {part}"
                continue
            b, r = p // 64, p % 64
            see = D.visible(1, p, p + 1, self.window, self.sinks)
            for h in range(self.h_kv):
                k = x[self.rq + h * dim: self.rq + (h + 1) * dim, c]
                k = D.rotated(k[None], [p], THETA)[0]
                v = x[self.rq + self.rk + h * dim: self.rq + self.rk + (h + 1) * dim, c]
                assert a["tail_block"][c, h] == b
                row = a["k_tail"][c, h, r].astype(np.float64)
                fine = np.isfinite(k)
                assert np.array_equal(np.isfinite(row), fine)
                assert np.all(np.abs(row - k)[fine] <= (D.HALF16 * np.abs(k) + 2.0 ** -22 * np.abs(k[fine]).max() + D.TINY16)[fine]), "the appended key"
                assert np.array_equal(a["v_tail"][c, h, :, r], v.astype(np.float16), equal_nan=True), "the appended value"
                if before["tail_block"][c, h] == b:
                    assert np.array_equal(a["k_tail"][c, h, :r], before["k_tail"][c, h, :r], equal_nan=True) and np.array_equal(a["v_tail"][c, h, :, :r], before["v_tail"][c, h, :, :r], equal_nan=True)
                else:                                               # back in a block that was complete: its 8-bit values
                    bk, bv = block_values(before, c, h, b, dim)
                    assert np.all(np.abs(a["k_tail"][c, h, :r] - bk[:r]) <= (D.HALF16 + 2.0 ** -23) * np.abs(bk[:r]) + D.TINY16)
                    assert np.all(np.abs(a["v_tail"][c, h, :, :r].T - bv[:r]) <= (D.HALF16 + 2.0 ** -23) * np.abs(bv[:r]) + D.TINY16)
                blocks = [block_values(before, c, h, i, dim) for i in range(b)]
                K = np.concatenate([i[0] for i in blocks] + [a["k_tail"][c, h, : r + 1].astype(np.float64)])
                V = np.concatenate([i[1] for i in blocks] + [a["v_tail"][c, h, :, : r + 1].astype(np.float64).T])
                q = D.rotated(x[h * g * dim: (h + 1) * g * dim, c].reshape(g, dim), [p] * g, THETA)
                # q is held as two FP16 numbers (2^-21), scores in 32 bits
                want, bound = D.attend(q, K, V, np.repeat(see, g, 0), 2.0 ** -21 + dim * 2.0 ** -23)
                within(out[h * g * dim: (h + 1) * g * dim, c].reshape(g, dim), want, bound, f"column {c} head {h} position {p}")
                other = np.ones(a["codes"].shape[2], dtype=bool)
                if r == 63:
                    check_block(a, c, h, b, a["k_tail"][c, h].astype(np.float64), a["v_tail"][c, h].astype(np.float64).T, "a completed block")
                    other[b] = False
                assert np.array_equal(a["codes"][c, h][other], before["codes"][c, h][other]) and np.array_equal(a["scales"][c, h][other], before["scales"][c, h][other], equal_nan=True), "other blocks stay"


@pytest.mark.parametrize("h_q,h_kv,dim,window,sinks", [(4, 1, 64, 0, 0), (8, 1, 64, 70, 3), (2, 2, 128, 0, 0), (9, 1, 64, 0, 0), (16, 1, 128, 130, 65), (3, 1, 128, 1, 0),
                                                       (16, 2, 64, 64, 64), (1, 1, 64, 200, 1000), (12, 1, 128, 0, 0), (5, 5, 64, 100, 0)])
def test_kv8_attention(h_q, h_kv, dim, window, sinks):
    positions = np.array([0, 1, 62, 63, 64, 65, 126, 127, 128, 200, 319, -1, 250], dtype=np.int32)
    d = Decoder(h_q, h_kv, dim, positions.size, 320, window, sinks, seed=h_q * dim + window)
    d.history()
    first = d.step(positions)
    again = d.step(positions, graph=True, tag=False, body=d.body)
    assert np.array_equal(first.view(np.uint16), again.view(np.uint16)), "the same step again gives the same bits"
    d.step(np.roll(positions, 5), graph=True)
    d.step(np.full(positions.size, -1), graph=True)
    d.plan.close()


@pytest.mark.parametrize("h_q,h_kv,dim,columns,pos,window,sinks", [(4, 1, 64, 1, 5000, 0, 0), (8, 8, 64, 1, 1500, 0, 0), (4, 2, 128, 3, 4095, 0, 0), (2, 1, 64, 100, 300, 0, 0),
                                                                   (4, 1, 64, 2, 9000, 1000, 70), (32, 8, 64, 70, 130, 0, 0)])
def test_kv8_attention_sizes(h_q, h_kv, dim, columns, pos, window, sinks):
    """Work split over many warps (few columns), many columns per warp, and windows far from the start."""
    d = Decoder(h_q, h_kv, dim, columns, pos + 3, window, sinks, seed=pos)
    d.history()
    p = d.rng.integers(-1, pos + 1, columns)
    p[0] = pos
    d.step(p)
    p[p >= 0] += 1
    d.step(p)
    d.plan.close()


def test_kv8_attention_hidden_places_do_not_count():
    import torch
    d = Decoder(4, 1, 64, 4, 400, window=50, sinks=5, seed=77)
    d.history()
    v = d.cache.views()
    codes = v["codes"].view(torch.uint8)
    codes[:, :, 0, 0].view(4, 1, 64, 64)[:, :, 5:] = 0x7f           # keys behind the sinks
    codes[:, :, 0, 1].view(4, 1, 64, 64)[:, :, :, 5:] = 0xff        # values behind the sinks
    codes[:, :, 1] = 0x7f                                           # a block that nobody sees
    v["scales"][:, :, 1] = float("nan")
    codes[:, :, 3, 1].view(4, 1, 64, 64)[:, :, :, : 300 - 49 - 192] = 0x7f      # values before the window
    v["k_tail"][:, :, 300 % 64 + 1:] = float("nan")                 # rows behind the last token
    v["v_tail"][:, :, :, 300 % 64 + 1:] = float("inf")
    out = d.step([300, 300, 300, 300])
    assert np.isfinite(out).all()
    # what is seen does count
    codes[1, :, 0, 1].view(1, 64, 64)[:, 7, 2] = 0x7f               # dimension 7 of a sink's value
    body = d.body.copy()
    body[d.rq + d.rk + 11, 2] = np.inf                              # the new token's value
    body[3, 3] = np.nan                                             # one query
    out = d.step([300, 300, 300, 300], body=body)
    assert np.isnan(out[7, 1]) and out[11, 2] == np.inf and np.isnan(out[:64, 3]).all() and np.isfinite(out[64:, 3]).all()
    d.plan.close()


def test_kv8_attention_odd_values_survive_the_8_bits():
    """A block with an infinity, a NaN, zeros and tiny numbers, completed by a step and read by the next ones."""
    import torch
    d = Decoder(1, 1, 64, 3, 200, seed=5)
    d.history()
    v = d.cache.views()
    v["k_tail"][0], v["v_tail"][0] = 0, 0
    v["v_tail"][1, 0, 3, 10], v["v_tail"][1, 0, 4, 11] = float("nan"), float("-inf")
    v["k_tail"][2], v["v_tail"][2] = 2.0 ** -24, 2.0 ** -24
    body = d.rng.normal(0, 1, (3 * 64, d.pitch)).astype(np.float16)
    body[64:, 0] = 0
    body[64:, 2] = np.float16(2.0 ** -24)
    d.step([63, 63, 63], body=body)
    codes = v["codes"].view(torch.uint8)[1, 0, 0, 1].view(64, 64).cpu().numpy()
    assert (codes[3, 10] & 0x7f) == 0x7f and codes[4, 11] == 0xfe and not (codes[3, 11] & 0x7f) == 0x7f
    d.step([64, 64, 64], tag=False)
    d.plan.close()


def test_kv8_positions_may_go_back():
    d = Decoder(2, 1, 64, 2, 256, seed=6)
    d.history()
    for p in range(60, 70):                        # over a block's end
        d.step([p, p + 64], tag=p == 60)
    d.step([40, 40], tag=False)                    # into a complete block
    d.step([41, -1], tag=False)
    d.step([0, 41], tag=False)                     # a new sequence, and on
    d.step([1, 42], tag=False)
    d.plan.close()


def test_kv8_position_outside_the_cache_is_reported():
    d = Decoder(2, 1, 64, 2, 100, seed=8)
    with pytest.raises(NativeError):
        d.plan.set_positions([100, 0])
    with pytest.raises(NativeError):
        d.plan.set_positions([-2, 0])
    with pytest.raises(NativeError):
        d.plan.set_positions([0, 0, 0])
    d.plan.close()


def test_prompt_then_tokens_then_answers():
    """As they are used together: a prompt plan with attention and fill, then a decode plan that starts from its cache: attention, a dense
    wave for the logits, probabilities, and a greedy arg-max that moves the positions on."""
    import torch
    from snntome_b200.plan import Wave
    h_q, h_kv, dim, seq, frames, window, sinks = 4, 2, 64, 150, 3, 90, 4
    rng = np.random.default_rng(12)
    rq, rk, cols = h_q * dim, h_kv * dim, frames * seq
    lengths = np.array([150, 64, 1], dtype=np.int32)
    slots = np.array([2, 0, 1], dtype=np.int32)
    cache = KV8Cache(4, h_kv, dim, 300)
    pitch = pitch_of(cols)
    prompt = rng.normal(0, 1, (rq + 2 * rk, pitch)).astype(np.float16)
    pp, pc = make_plan(prompt, rq, cols)
    pp.add_window_attn(0, rq * pitch, (rq + rk) * pitch, (rq + 2 * rk) * pitch, h_q, h_kv, dim, seq, window=window, sinks=sinks, theta=THETA)
    pp.add_kv8_fill(cache, rq * pitch, (rq + rk) * pitch, seq, theta=THETA)
    pp.set_sequences(slots, lengths)
    pp.execute_graph()
    assert pp.status() == 0
    x = prompt[:, :cols].astype(np.float64)
    want, bound = D.window_attention(x[:rq], x[rq: rq + rk], x[rq + rk:], h_q, h_kv, seq, cols, window, sinks, THETA)
    within(read(pc, pitch)[rq + 2 * rk:, :cols], want, bound, "prompt")

    vocab, columns = 512, 4
    d = Decoder(h_q, h_kv, dim, columns, 300, window, sinks, seed=13, cache=cache)
    body = d.rng.normal(0, 1, (rq + 2 * rk, d.pitch)).astype(np.float16)
    total = (2 * rq + 2 * rk + vocab) * d.pitch
    plan = NativePlan.create(total, d.pitch, columns)
    canvas = plan.canvas_tensor()
    p = d.pitch
    out_off = (rq + 2 * rk) * p
    plan.add_kv8_attn(cache, 0, rq * p, (rq + rk) * p, out_off, h_q, window=window, sinks=sinks, theta=THETA)
    w = rng.normal(0, 0.3, (vocab, rq)).astype(np.float16)
    idx = (np.arange(rq, dtype=np.uint32) * p + out_off)[None, :].repeat(vocab // 128, axis=0)
    plan.add_wave(Wave(cout=vocab, group=128, fan_in=rq, idx=idx, weights=w.view(np.uint16), bias=None, y_off=out_off + rq * p, act=0, name="head"))
    t = dict(targets=torch.arange(columns, dtype=torch.int32, device="cuda"), logprobs=torch.empty(columns, device="cuda"), entropy=torch.empty(columns, device="cuda"),
             top_rows=torch.empty(3, columns, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(3, columns, device="cuda"))
    plan.add_argmax(out_off + rq * p, vocab, advance=True, max_seq=300)
    plan.add_logprobs(out_off + rq * p, vocab, **t)
    positions = np.full(columns, -1, dtype=np.int32)
    positions[slots] = lengths
    plan.set_positions(positions)
    d.plan, d.canvas = plan, canvas
    for step in range(4):
        canvas[: body.size] = torch.from_numpy(body.reshape(-1)).cuda()
        before = cache_arrays(cache)
        plan.execute_graph()
        assert plan.status() == 0
        got = read(canvas, p)
        d.check(positions, body, got[rq + 2 * rk: 2 * rq + 2 * rk, :columns], before, cache_arrays(cache))
        logits = got[2 * rq + 2 * rk:, :columns].astype(np.float64)
        lp, ent = D.logprobs(logits)
        assert np.array_equal(t["top_rows"].cpu().numpy(), D.top_rows(logits, 3))
        assert np.array_equal(t["top_rows"].cpu().numpy()[0], plan.next_tokens(columns))
        assert np.allclose(t["top_logprobs"].cpu().numpy(), np.take_along_axis(lp, D.top_rows(logits, 3), 0), rtol=2.0 ** -21, atol=8e-6)
        assert np.allclose(t["logprobs"].cpu().numpy(), lp[np.arange(columns), np.arange(columns)], rtol=2.0 ** -21, atol=8e-6)
        positions[positions >= 0] += 1             # as the arg-max did on the device
        body = d.rng.normal(0, 1, body.shape).astype(np.float16)
    plan.close()
    pp.close()


# ---- answers ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,columns,top", [(1, 1, 1), (2, 9, 2), (63, 3, 5), (64, 64, 32), (65, 17, 32), (513, 40, 7), (1000, 100, 0), (5000, 30, 32), (33, 70, 32), (128 * 64 + 1, 1, 32),
                                              (140000, 2, 20)])
def test_logprobs(rows, columns, top):
    import torch
    rng = np.random.default_rng(rows + columns)
    pitch = pitch_of(columns)
    x = (rng.normal(0, 3, (rows, pitch)) if rows % 2 else rng.integers(-20, 20, (rows, pitch)) / 4.0).astype(np.float16)     # even: plenty of ties
    if rows > 60:
        x[rng.random(rows) < 0.2] = -np.inf
        x[rows // 2, ::3] = np.float16(-0.0)
        x[rows // 2 + 1, ::3] = np.float16(0.0)
        x[3, :] = np.float16(-65504)
    x[-1] = 1.0
    x[:, columns:] = np.nan
    if columns > 8:
        x[:, 1] = -np.inf
        x[rows // 2, 2] = np.nan
        x[0, 3] = np.inf
        x[:, 4] = np.nan
        x[:, 5] = np.float16(65504)
    plan, canvas = make_plan(x, 0, columns)
    targets = rng.integers(0, rows, columns).astype(np.int32)
    targets[-1] = rows if columns > 2 else 0
    if columns > 10:
        targets[9] = -1
    f = lambda *s: torch.full(s, -5.0, device="cuda")
    t = dict(targets=torch.from_numpy(targets).cuda(), logprobs=f(columns), entropy=f(columns))
    if top:
        t.update(top_rows=torch.full((top, columns), -5, dtype=torch.int32, device="cuda"), top_logprobs=f(top, columns))
    plan.add_logprobs(0, rows, **t)
    for run in (plan.execute, plan.execute_graph):
        run()
        assert plan.status() == 0
        y = x[:, :columns].astype(np.float64)
        lp, ent = D.logprobs(y)
        want = np.where((targets >= 0) & (targets < rows), lp[targets.clip(0, rows - 1), np.arange(columns)], np.nan)
        # the sum is good to 2^-18 (exponentials of up to 12 effective nats and a tree of about 40 additions, 2^-24 each), the rest to 32 bits
        tol = lambda v: 2.0 ** -18 + 2.0 ** -21 * np.abs(np.where(np.isfinite(v), v, 0.0))
        within(t["logprobs"].cpu().numpy(), want, tol(want), "log probability")
        within(t["entropy"].cpu().numpy(), ent, 2.0 ** -17 + 2.0 ** -16 * np.abs(np.where(np.isfinite(ent), ent, 0.0)) + 2.0 ** -16 * np.log(rows + 1), "entropy")
        if top:
            best = D.top_rows(y, top)
            assert np.array_equal(t["top_rows"].cpu().numpy(), best)
            bl = np.take_along_axis(lp, best, 0)
            within(t["top_logprobs"].cpu().numpy(), bl, tol(bl), "alternatives")
    plan.close()


# ---- refusals --------------------------------------------------------------------------------------------------------------------------
def test_refusals():
    import torch
    plan = NativePlan.create(640 * 64, 64, 50)
    cache = KV8Cache(50, 1, 64, 100)
    ok = dict(q_off=0, k_off=64 * 64, v_off=128 * 64, out_off=192 * 64, h_q=1, h_kv=1, head_dim=64, seq_len=50)
    for bad in [dict(head_dim=96), dict(h_q=0), dict(h_kv=0), dict(h_q=3, h_kv=2), dict(seq_len=0), dict(out_off=0), dict(out_off=63 * 64), dict(q_off=4), dict(v_off=600 * 64),
                dict(theta=0.0), dict(theta=float("nan")), dict(window=-1), dict(sinks=1 << 31), dict(q_off=-64), dict(k_off=1 << 62)]:
        with pytest.raises(NativeError):
            plan.add_window_attn(**{**ok, **bad})
    ok = dict(cache=cache, k_off=0, v_off=64 * 64, seq_len=10)
    for bad in [dict(k_off=639 * 64), dict(seq_len=0), dict(v_off=3), dict(theta=1.0)]:
        with pytest.raises(NativeError):
            plan.add_kv8_fill(**{**ok, **bad})
    ok = dict(cache=cache, q_off=0, k_off=64 * 64, v_off=128 * 64, out_off=192 * 64, h_q=1)
    for bad in [dict(cache=KV8Cache(49, 1, 64, 100)), dict(h_q=0), dict(h_q=17), dict(out_off=64 * 64), dict(q_off=620 * 64), dict(cache=KV8Cache(50, 3, 64, 100), h_q=4)]:
        with pytest.raises(NativeError):
            plan.add_kv8_attn(**{**ok, **bad})
    for bad in [torch.empty(10, dtype=torch.uint8, device="cuda"), torch.empty(1 << 24, dtype=torch.uint8), torch.empty(1 << 24, dtype=torch.uint8, device="cuda")[8:]]:
        with pytest.raises(NativeError):
            KV8Cache(50, 1, 64, 100, storage=bad)
    f = torch.empty(50, device="cuda")
    i = torch.zeros(50, dtype=torch.int32, device="cuda")
    for bad in [dict(), dict(targets=i), dict(logprobs=f), dict(entropy=f[:10]), dict(entropy=f.double()), dict(entropy=f.cpu()), dict(targets=i.long(), logprobs=f),
                dict(top_rows=torch.zeros(2, 50, dtype=torch.int32, device="cuda")), dict(rows=641, entropy=f), dict(rows=0, entropy=f), dict(src_off=1, entropy=f),
                dict(top_rows=torch.zeros(33, 50, dtype=torch.int32, device="cuda"), top_logprobs=torch.zeros(33, 50, device="cuda")),
                dict(rows=2, top_rows=torch.zeros(3, 50, dtype=torch.int32, device="cuda"), top_logprobs=torch.zeros(3, 50, device="cuda"))]:
        with pytest.raises(NativeError):
            plan.add_logprobs(**{**dict(src_off=0, rows=100), **bad})
    assert plan.num_waves == 0
    plan.add_kv8_fill(cache, 0, 64 * 64, 10)
    for slots, lengths in [([0, 0], [1, 1]), ([50], [1]), ([0], [11]), ([0], [-1]), ([-2], [1]), ([0], [1, 2]), (list(range(6)), [10, 10, 10, 10, 10, 1])]:
        with pytest.raises(NativeError):
            plan.set_sequences(slots, lengths)
    plan.set_sequences([-1, 3, -1], [99, 10, 0])
    with pytest.raises(NativeError):
        plan.add_kv8_fill(KV8Cache(3, 1, 64, 100), 0, 64 * 64, 10)         # the sequences set before do not fit it
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        with pytest.raises(NativeError):
            plan.set_sequences([-1], [0], stream=s)
        with pytest.raises(NativeError):
            plan.set_positions([-1], stream=s)
        torch.zeros(1, device="cuda")
    plan.execute()
    assert plan.status() == 0
    plan.close()
