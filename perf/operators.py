"""The attention, cache and answer operators of a decoder as measured cases: what a case stands for, its inputs, its plain form
in elementary torch operations, and its definition in 64 bits.

Four operators, each a command of a plan (`snntome_b200.native.NativePlan`):

* `window_attn`  prompts: rotary embedding and causal grouped-query attention with a sliding window and sinks
* `kv8_fill`     prompts: keys and values into a cache of 8 bits with one scale per block of 64 tokens, head and column
* `kv8_attn`     single tokens: append to that cache and attend to it, every column at a position of its own
* `logprobs`     log probability of a given token, entropy and top alternatives per column of a logits tensor

Tensors on the canvas are channel-major FP16: channel c of a tensor at element offset `off` is canvas[off + c*pitch ...].
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64              # tokens per block of the 8-bit cache
THETA = 500000.0        # rotary base of the decoder whose shapes the benchmark uses
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a short chat turn as a prompt: one sequence of odd length, where launches count
        dict(name="prompt-100", op="window_attn", frames=1, seq=100, h_q=32, h_kv=8, dim=64, window=0, sinks=0),
        # four prompts of 1000 tokens, 128 dimensions per head: full causal attention, sequences that end inside tiles
        dict(name="prompts-4x1000-d128", op="window_attn", frames=4, seq=1000, h_q=32, h_kv=8, dim=128, window=0, sinks=0),
        # one long prompt of a model with a window of 1024 tokens and 4 sinks
        dict(name="prompt-8192-window", op="window_attn", frames=1, seq=8192, h_q=32, h_kv=8, dim=64, window=1024, sinks=4),
        # a single prompt of 200 tokens into the cache of one layer
        dict(name="fill-200", op="kv8_fill", frames=1, seq=200, h_kv=8, dim=64, columns=4, max_seq=1024, ragged=0),
        # a batch of 64 prompts of up to 512 tokens (the benchmark's decoder: 64 columns, 512 positions)
        dict(name="fill-64x512", op="kv8_fill", frames=64, seq=512, h_kv=8, dim=64, columns=64, max_seq=1024, ragged=1),
        # one sequence alone: the latency of a single user's token
        dict(name="token-1x1500", op="kv8_attn", columns=1, pos=1500, ragged=0, h_q=32, h_kv=8, dim=64, max_seq=4096, window=0, sinks=0),
        # the benchmark's decoder step: 64 sequences at 511 cached positions; the step's token completes a block
        dict(name="tokens-64x512", op="kv8_attn", columns=64, pos=511, ragged=0, h_q=32, h_kv=8, dim=64, max_seq=512, window=0, sinks=0),
        # 48 sequences of mixed lengths up to 8192, 128 dimensions per head, some columns idle
        dict(name="tokens-48x8192-d128", op="kv8_attn", columns=48, pos=8190, ragged=1, h_q=32, h_kv=8, dim=128, max_seq=8192, window=0, sinks=0),
        # 64 long sequences of a model with a window of 1024 tokens and 4 sinks
        dict(name="tokens-64x16384-window", op="kv8_attn", columns=64, pos=16000, ragged=1, h_q=32, h_kv=8, dim=64, max_seq=16384, window=1024, sinks=4),
        # one sequence's next-token probabilities
        dict(name="answer-1", op="logprobs", rows=128256, columns=1, top=5),
        # a decode step of the benchmark's decoder: 64 sequences with 20 alternatives each
        dict(name="answers-64", op="logprobs", rows=128256, columns=64, top=20),
        # scoring the tokens of a prompt of 1000
        dict(name="score-1000", op="logprobs", rows=128256, columns=1000, top=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window_attn", "kv8_fill", "kv8_attn", "logprobs"])
    h_kv = rng.choice([1, 2, 4, 8])
    h_q = h_kv * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128])
    if op == "window_attn":
        most = min(8192, 8192 * 32 * 64 // (h_q * dim))          # tokens
        window = rng.choice([0, _log(rng, 1, 1024)])
        seq = _log(rng, 1, most if window else min(most, 2000))
        frames = _log(rng, 1, max(1, min(64, most // seq)))
        return dict(op=op, frames=frames, seq=seq, h_q=h_q, h_kv=h_kv, dim=dim, window=window, sinks=rng.choice([0, 1, 4, 100]))
    if op == "kv8_fill":
        most = min(32768, 64 * 512 * 8 * 64 // (h_kv * dim))
        seq = _log(rng, 1, 4096)
        frames = _log(rng, 1, max(1, min(64, most // seq)))
        return dict(op=op, frames=frames, seq=seq, h_kv=h_kv, dim=dim, columns=frames + rng.randrange(3), max_seq=seq + rng.randrange(200), ragged=rng.choice([0, 1]))
    if op == "kv8_attn":
        pos = _log(rng, 1, 16384) - 1
        columns = _log(rng, 1, max(1, min(64, 24 * 8192 * 8 * 128 // (h_kv * dim * (pos + 1)))))
        return dict(op=op, columns=columns, pos=pos, ragged=rng.choice([0, 1]), h_q=h_q, h_kv=h_kv, dim=dim, max_seq=pos + 1 + rng.randrange(300),
                    window=rng.choice([0, _log(rng, 1, 4096)]), sinks=rng.choice([0, 1, 4, 100]))
    rows = _log(rng, 2, 128256)
    return dict(op=op, rows=rows, columns=_log(rng, 1, 1000), top=rng.randrange(0, min(rows, 32) + 1))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pitch(columns):
    return (columns + 63) // 64 * 64


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(torch.float16)


def _up256(n):
    return (n + 255) // 256 * 256


def cache_bytes(columns, h_kv, dim, max_seq):
    nb = (max_seq + BLOCK - 1) // BLOCK
    ch = columns * h_kv
    return _up256(ch * nb * 2 * BLOCK * dim) + _up256(ch * nb * 8) + 2 * _up256(ch * BLOCK * dim * 2) + _up256(ch * 4)


def cache_views(storage, columns, h_kv, dim, max_seq):
    """The parts of an 8-bit cache in its storage: codes of K as [column][head][block][dim / 64][token][64], of V as
    [column][head][block][dim][token] (side by side per block), scales [column][head][block][K, V], the FP16 rows of the
    open block of K [column][head][token][dim] and of V [column][head][dim][token], and the number of that block."""
    nb = (max_seq + BLOCK - 1) // BLOCK
    ch = columns * h_kv
    at = 0

    def part(n, dtype):
        nonlocal at
        v = storage[at: at + n].view(dtype)
        at += _up256(n)
        return v

    codes = part(ch * nb * 2 * BLOCK * dim, E4M3).view(columns, h_kv, nb, 2, BLOCK * dim)
    scales = part(ch * nb * 8, torch.float32).view(columns, h_kv, nb, 2)
    k_tail = part(ch * BLOCK * dim * 2, torch.float16).view(columns, h_kv, BLOCK, dim)
    v_tail = part(ch * BLOCK * dim * 2, torch.float16).view(columns, h_kv, dim, BLOCK)
    tail_block = part(ch * 4, torch.int32).view(columns, h_kv)
    return dict(codes=codes, scales=scales, k_tail=k_tail, v_tail=v_tail, tail_block=tail_block)


def _k_to_codes(x):      # [..., token, dim] -> [..., dim / 64 * token * 64]
    d = x.shape[-1]
    return x.unflatten(-1, (d // 64, 64)).transpose(-3, -2).flatten(-3)


def _k_from_codes(x, dim):
    return x.unflatten(-1, (dim // 64, BLOCK, 64)).transpose(-3, -2).flatten(-2)


def _quantise(x):
    """x: FP32 values of FP16 numbers [..., token, dim] -> (codes, scale): one scale per block."""
    scale = x.abs().amax(dim=(-2, -1)).clamp_min(2.0 ** -24) / 448.0
    return (x / scale[..., None, None]).to(E4M3), scale


def _history(g, case, views):
    """A cache that holds earlier positions: keys with a few strong channels, as rotated keys have them, and values."""
    c, h, nb = views["codes"].shape[:3]
    d = case["dim"]
    loud = torch.ones(d, device="cuda")
    loud[torch.randperm(d, generator=g, device="cuda")[: d // 16]] = 4.0
    x = torch.randn(c, h, nb, BLOCK, d, generator=g, device="cuda").mul_(loud).half().float()
    codes, scale = _quantise(x)
    views["codes"].view(torch.uint8)[:, :, :, 0] = _k_to_codes(codes.view(torch.uint8))
    views["scales"][..., 0] = scale
    x = torch.randn(c, h, nb, BLOCK, d, generator=g, device="cuda").half().float()
    codes, scale = _quantise(x)
    views["codes"].view(torch.uint8)[:, :, :, 1] = codes.view(torch.uint8).transpose(-2, -1).flatten(-2)
    views["scales"][..., 1] = scale
    views["k_tail"].copy_(torch.randn(views["k_tail"].shape, generator=g, device="cuda") * loud)
    views["v_tail"].copy_(torch.randn(views["v_tail"].shape, generator=g, device="cuda"))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case=case)
    if op == "window_attn":
        cols = case["frames"] * case["seq"]
        pitch = _pitch(cols)
        d, hq, hk = case["dim"], case["h_q"], case["h_kv"]
        rows = 2 * (hq + hk) * d                         # q, k, v, out
        s["canvas"] = torch.zeros(rows * pitch, dtype=torch.float16, device="cuda")
        s["canvas"][: (hq + 2 * hk) * d * pitch] = _normal(g, (hq + 2 * hk) * d * pitch)
        s.update(pitch=pitch, cols=cols, q=0, k=hq * d * pitch, v=(hq + hk) * d * pitch, out=(hq + 2 * hk) * d * pitch)
    elif op == "kv8_fill":
        cols = case["frames"] * case["seq"]
        pitch = _pitch(cols)
        d, hk, n = case["dim"], case["h_kv"], case["frames"]
        s["canvas"] = _normal(g, 2 * hk * d * pitch)
        s.update(pitch=pitch, cols=cols, k=0, v=hk * d * pitch)
        s["lengths"] = torch.randint(0, case["seq"] + 1, (n,), generator=g, device="cuda") if case["ragged"] else torch.full((n,), case["seq"], device="cuda")
        s["slots"] = torch.randperm(case["columns"], generator=g, device="cuda")[:n]
        s["storage"] = torch.zeros(cache_bytes(case["columns"], hk, d, case["max_seq"]), dtype=torch.uint8, device="cuda")
        s["cache"] = cache_views(s["storage"], case["columns"], hk, d, case["max_seq"])
        s["cache"]["tail_block"].fill_(-1)
    elif op == "kv8_attn":
        cols = case["columns"]
        pitch = _pitch(cols)
        d, hq, hk = case["dim"], case["h_q"], case["h_kv"]
        s["canvas"] = torch.zeros(2 * (hq + hk) * d * pitch, dtype=torch.float16, device="cuda")
        s["canvas"][: (hq + 2 * hk) * d * pitch] = _normal(g, (hq + 2 * hk) * d * pitch)
        s.update(pitch=pitch, cols=cols, q=0, k=hq * d * pitch, v=(hq + hk) * d * pitch, out=(hq + 2 * hk) * d * pitch)
        s["storage"] = torch.zeros(cache_bytes(cols, hk, d, case["max_seq"]), dtype=torch.uint8, device="cuda")
        s["cache"] = cache_views(s["storage"], cols, hk, d, case["max_seq"])
        _history(g, case, s["cache"])
        pos = torch.randint(-1, case["pos"] + 1, (cols,), generator=g, device="cuda") if case["ragged"] else torch.full((cols,), case["pos"], device="cuda")
        pos[0] = case["pos"]
        s["pos"] = pos
        # the open block is that of the position before
        s["cache"]["tail_block"].copy_(torch.where(pos > 0, (pos - 1).clamp_min(0) // BLOCK, -1)[:, None].expand(cols, hk))
    else:
        cols, rows = case["columns"], case["rows"]
        pitch = _pitch(cols)
        x = torch.randn(rows, pitch, generator=g, device="cuda").mul_(3.0)
        x[torch.rand(rows, generator=g, device="cuda") < 0.01] = -math.inf          # tokens that must not be answered
        x[rows - 1] = 1.0
        s["canvas"] = x.to(torch.float16).reshape(-1)
        del x
        s.update(pitch=pitch, cols=cols)
        s["targets"] = torch.randint(0, rows, (cols,), generator=g, device="cuda", dtype=torch.int32)
        banned = torch.isinf(s["canvas"].view(rows, pitch)[:, 0])[s["targets"].long()]
        s["targets"][banned] = rows - 1
        top = case["top"]
        s["out"] = (torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda"), torch.empty(top, cols, dtype=torch.int32, device="cuda"), torch.empty(top, cols, device="cuda"))
    if own:
        _build(s)
    return s


def _build(s):
    """The plan that a user's program keeps: one command over its canvas."""
    from snntome_b200.native import KV8Cache, NativePlan
    case = s["case"]
    plan = s["plan"] = NativePlan.create(s["canvas"].numel(), s["pitch"], s["cols"])
    canvas = plan.canvas_tensor()
    canvas.copy_(s["canvas"])
    s["canvas"] = canvas
    if case["op"] == "window_attn":
        plan.add_window_attn(s["q"], s["k"], s["v"], s["out"], case["h_q"], case["h_kv"], case["dim"], case["seq"], window=case["window"], sinks=case["sinks"], theta=THETA, llama3=False)
    elif case["op"] == "kv8_fill":
        cache = KV8Cache(case["columns"], case["h_kv"], case["dim"], case["max_seq"], storage=s["storage"])
        plan.add_kv8_fill(cache, s["k"], s["v"], case["seq"], theta=THETA, llama3=False)
        s["sequences"] = s["slots"].cpu().numpy(), s["lengths"].cpu().numpy()          # what a scheduler has on the host
    elif case["op"] == "kv8_attn":
        cache = KV8Cache(case["columns"], case["h_kv"], case["dim"], case["max_seq"], storage=s["storage"])
        plan.add_kv8_attn(cache, s["q"], s["k"], s["v"], s["out"], case["h_q"], window=case["window"], sinks=case["sinks"], theta=THETA, llama3=False)
        s["positions"] = s["pos"].cpu().numpy()
    else:
        lp, ent, rows, tlp = s["out"]
        plan.add_logprobs(0, case["rows"], s["targets"], lp, ent, rows, tlp)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        # where the pass's sequences go and what its tokens' positions are come with every pass
        if op == "kv8_fill":
            s["plan"].set_sequences(*s["sequences"])
        elif op == "kv8_attn":
            s["plan"].set_positions(s["positions"])
        s["plan"].execute()
    elif op == "window_attn":
        _plain_window_attn(s)
    elif op == "kv8_fill":
        _plain_fill(s)
    elif op == "kv8_attn":
        _plain_kv8_attn(s)
    else:
        return _plain_logprobs(s)
    if op == "kv8_fill":
        return dict(s["cache"])
    if op == "logprobs":
        lp, ent, rows, tlp = s["out"]
        return dict(logprobs=lp, entropy=ent, top_rows=rows, top_logprobs=tlp)
    out = s["canvas"][s["out"]:].view(case["h_q"] * case["dim"], s["pitch"])[:, : s["cols"]]
    return dict(out=out, **s["cache"]) if op == "kv8_attn" else dict(out=out)


def _rows(s, off, n):
    return s["canvas"][off: off + n * s["pitch"]].view(n, s["pitch"])[:, : s["cols"]]


def _rotate(x, pos):
    """x [..., dim] in 32 bits at positions pos (broadcastable to x's leading axes): pairs (p, p + dim / 2)."""
    half = x.shape[-1] // 2
    freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 * math.log(THETA) / x.shape[-1]))
    ang = pos[..., None].double() * freq
    c, n = torch.cos(ang).float(), torch.sin(ang).float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * n, a * n + b * c], dim=-1)


def _visible(t, c, window, sinks):
    see = c <= t
    return see if window == 0 else see & ((c > t - window) | (c < sinks))


def _plain_window_attn(s):
    case = s["case"]
    d, hq, hk, f, n = case["dim"], case["h_q"], case["h_kv"], case["frames"], case["seq"]
    pos = torch.arange(n, device="cuda")

    def heads(off, h):       # [frame, head, token, dim]
        return _rows(s, off, h * d).float().view(h, d, f, n).permute(2, 0, 3, 1)

    q = _rotate(heads(s["q"], hq), pos)
    k = _rotate(heads(s["k"], hk), pos)
    v = heads(s["v"], hk)
    sc = torch.matmul(q.reshape(f, hk, -1, d), k.transpose(-2, -1)).view(f, hq, n, n).div_(math.sqrt(d))
    sc.masked_fill_(~_visible(pos[:, None], pos[None, :], case["window"], case["sinks"]), -math.inf)
    sc.sub_(sc.amax(dim=-1, keepdim=True)).exp_()
    total = sc.sum(dim=-1, keepdim=True)
    o = torch.matmul(sc.view(f, hk, -1, n), v).view(f, hq, n, d) / total
    _rows(s, s["out"], hq * d).copy_(o.permute(1, 3, 0, 2).reshape(hq * d, f * n))


def _plain_fill(s):
    case = s["case"]
    d, hk, f, n = case["dim"], case["h_kv"], case["frames"], case["seq"]
    nb = s["cache"]["codes"].shape[2]
    room = nb * BLOCK
    pos = torch.arange(n, device="cuda")
    k = _rows(s, s["k"], hk * d).float().view(hk, d, f, n).permute(2, 0, 3, 1)
    v = _rows(s, s["v"], hk * d).float().view(hk, d, f, n).permute(2, 0, 3, 1)
    k = _rotate(k, pos).half().float()
    pad = (0, 0, 0, room - n)
    k = torch.nn.functional.pad(k, pad).view(f, hk, nb, BLOCK, d)
    v = torch.nn.functional.pad(v, pad).view(f, hk, nb, BLOCK, d)
    slots, lengths = s["slots"], s["lengths"]
    full = (torch.arange(nb, device="cuda") < (lengths // BLOCK)[:, None])[:, None, :, None]          # [frame, 1, block, 1]
    c = s["cache"]
    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    codes = torch.stack([_k_to_codes(kc.view(torch.uint8)), vc.view(torch.uint8).transpose(-2, -1).flatten(-2)], dim=-2)
    raw = c["codes"].view(torch.uint8)
    raw[slots] = torch.where(full[..., None], codes, raw[slots])
    c["scales"][slots] = torch.where(full, torch.stack([ks, vs], dim=-1), c["scales"][slots])
    open_block = (lengths // BLOCK).clamp_max(nb - 1)
    rest = lengths % BLOCK
    at = open_block[:, None, None, None, None].expand(f, hk, 1, BLOCK, d)
    live = (torch.arange(BLOCK, device="cuda") < rest[:, None])[:, None, :, None]
    c["k_tail"][slots] = torch.where(live, k.gather(2, at)[:, :, 0].half(), c["k_tail"][slots])
    c["v_tail"][slots] = torch.where(live.transpose(-2, -1), v.gather(2, at)[:, :, 0].half().transpose(-2, -1), c["v_tail"][slots])
    c["tail_block"][slots] = torch.where(rest > 0, open_block, -1)[:, None].to(torch.int32).expand(f, hk)


def _plain_kv8_attn(s):
    case, cache, pos = s["case"], s["cache"], s["pos"]
    d, hq, hk, cols = case["dim"], case["h_q"], case["h_kv"], s["cols"]
    nb = cache["codes"].shape[2]
    live = pos >= 0
    at = pos.clamp_min(0)
    q = _rotate(_rows(s, s["q"], hq * d).float().view(hq, d, cols).permute(2, 0, 1), at[:, None])
    k = _rotate(_rows(s, s["k"], hk * d).float().view(hk, d, cols).permute(2, 0, 1), at[:, None]).half()
    v = _rows(s, s["v"], hk * d).view(hk, d, cols).permute(2, 0, 1)
    # append the token to the open block
    col = torch.arange(cols, device="cuda")
    block, slot = at // BLOCK, at % BLOCK
    cache["k_tail"][col, :, slot] = torch.where(live[:, None, None], k, cache["k_tail"][col, :, slot])
    cache["v_tail"][col, :, :, slot] = torch.where(live[:, None, None], v, cache["v_tail"][col, :, :, slot])
    cache["tail_block"].copy_(torch.where(live[:, None], block[:, None].to(torch.int32), cache["tail_block"]))
    # attend: earlier blocks in 8 bits, the open one in FP16
    tok = torch.arange(nb * BLOCK, device="cuda")
    k8 = (_k_from_codes(cache["codes"][:, :, :, 0].float(), d) * cache["scales"][..., 0, None, None]).view(cols, hk, -1, d)
    v8 = (cache["codes"][:, :, :, 1].float().unflatten(-1, (d, BLOCK)) * cache["scales"][..., 1, None, None]).transpose(-2, -1).reshape(cols, hk, -1, d)
    qg = q.reshape(cols, hk, -1, d)
    sc = torch.cat([torch.matmul(qg, k8.transpose(-2, -1)), torch.matmul(qg, cache["k_tail"].float().transpose(-2, -1))], dim=-1) / math.sqrt(d)
    seen8 = _visible(at[:, None], tok[None], case["window"], case["sinks"]) & (tok[None] < (block * BLOCK)[:, None])
    seen16 = _visible(at[:, None], (block * BLOCK)[:, None] + tok[None, :BLOCK], case["window"], case["sinks"])
    sc.masked_fill_(~torch.cat([seen8, seen16], dim=-1)[:, None, None, :], -math.inf)
    sc.sub_(sc.amax(dim=-1, keepdim=True)).exp_()
    total = sc.sum(dim=-1, keepdim=True)
    o = (torch.matmul(sc[..., : nb * BLOCK], v8) + torch.matmul(sc[..., nb * BLOCK:], cache["v_tail"].float().transpose(-2, -1))) / total
    o = torch.where(live[:, None, None, None], o, 0.0)
    _rows(s, s["out"], hq * d).copy_(o.reshape(cols, hq * d).t())
    # a block whose last token has come is brought to 8 bits
    done = (live & (slot == BLOCK - 1))[:, None]
    kc, ks = _quantise(cache["k_tail"].float())
    vc, vs = _quantise(cache["v_tail"].float())
    raw = cache["codes"].view(torch.uint8)
    new = torch.stack([_k_to_codes(kc.view(torch.uint8)), vc.view(torch.uint8).flatten(-2)], dim=-2)
    raw[col, :, block] = torch.where(done[..., None, None], new, raw[col, :, block])
    cache["scales"][col, :, block] = torch.where(done[..., None], torch.stack([ks, vs], dim=-1), cache["scales"][col, :, block])


def _plain_logprobs(s):
    case, cols = s["case"], s["cols"]
    x16 = s["canvas"].view(case["rows"], s["pitch"])[:, :cols]
    x = x16.float()
    m = x.amax(dim=0)
    z = x - m
    p = z.exp()
    total = p.sum(dim=0)
    ln = total.log()
    entropy = ln - torch.where(p > 0, p * z, 0.0).sum(dim=0) / total
    lp = z.gather(0, s["targets"].long()[None])[0] - ln
    if case["top"] == 0:
        return dict(logprobs=lp, entropy=entropy, top_rows=s["out"][2], top_logprobs=s["out"][3])
    # by value, the lowest row first among equals: the value's order and the row in one whole number
    bits = x16.contiguous().view(torch.int16).to(torch.int64)
    order = torch.where(bits >= 0, bits, -(bits & 0x7fff))
    key = order * (1 << 32) + (case["rows"] - torch.arange(case["rows"], device="cuda"))[:, None]
    best = key.topk(case["top"], dim=0).values
    rows = case["rows"] - (best & 0xffffffff)
    return dict(logprobs=lp, entropy=entropy, top_rows=rows.to(torch.int32), top_logprobs=z.gather(0, rows) - ln)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _pairs(n, window, sinks):
    """Visible (query, key) pairs of a sequence of n tokens."""
    if window == 0 or window >= n:
        return n * (n + 1) // 2
    seen = window * (window + 1) // 2 + (n - window) * window
    seen += sum(min(sinks, t - window + 1) for t in range(window, min(n, window + sinks)))
    return seen + max(0, n - window - sinks) * min(sinks, n)


def work(case):
    op, d = case["op"], case.get("dim", 0)
    if op == "window_attn":
        t = case["frames"] * case["seq"]
        return dict(bytes=2.0 * 2 * (case["h_q"] + case["h_kv"]) * d * t, flops=4.0 * d * case["h_q"] * case["frames"] * _pairs(case["seq"], case["window"], case["sinks"]))
    share = 0.5 if case.get("ragged") else 1.0           # lengths spread evenly over the range
    if op == "kv8_fill":
        t = case["frames"] * case["seq"] * share
        return dict(bytes=t * 2 * case["h_kv"] * d * 3.0, flops=t * case["h_kv"] * d * 8.0)
    if op == "kv8_attn":
        n = (case["pos"] + 1) * share
        if case["window"]:
            n = min(n, case["window"] + case["sinks"])
        t = case["columns"] * n
        return dict(bytes=t * 2 * case["h_kv"] * d + case["columns"] * 2.0 * 2 * (case["h_q"] + case["h_kv"]) * d, flops=4.0 * t * case["h_q"] * d)
    return dict(bytes=2.0 * case["rows"] * case["columns"] + 8.0 * case["columns"] * (case["top"] + 2), flops=6.0 * case["rows"] * case["columns"])


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, written apart from the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _turn64(x, where):
    """x [dim, tokens] in 64 bits, tokens at positions `where`."""
    d = x.shape[0]
    p = torch.arange(d // 2, dtype=torch.float64, device=x.device)
    angle = (THETA ** (-2.0 * p / d))[:, None] * where.double()[None, :]
    top, low = x[: d // 2], x[d // 2:]
    return torch.cat((top * angle.cos() - low * angle.sin(), top * angle.sin() + low * angle.cos()), 0)


def _attend64(q, k, v, seen):
    """q [m, dim], k, v [n, dim], seen [m, n] -> [m, dim]"""
    w = (q @ k.t()) * q.shape[1] ** -0.5
    w = torch.softmax(torch.where(seen, w, torch.full_like(w, -math.inf)), dim=1)
    return w @ v


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    pitch = s["pitch"]
    tensor = lambda off, ch: s["canvas"][off: off + ch * pitch].view(ch, pitch).double()  # noqa: E731
    if op == "logprobs":
        n = case["rows"]
        lp, ent, tops = [], [], []
        allx = s["canvas"].view(n, pitch)
        for c0 in range(0, case["columns"], 64):
            x = allx[:, c0: min(c0 + 64, case["columns"])].double()
            logp = torch.log_softmax(x, dim=0)
            prob = torch.exp(logp)
            ent.append(-(prob * torch.where(prob > 0, logp, torch.zeros_like(logp))).sum(0))
            lp.append(logp.gather(0, s["targets"][c0: c0 + 64].long()[None])[0])
            tops.append(torch.sort(logp, dim=0, descending=True).values[: case["top"]] if case["top"] else logp[:0])
        # which rows they are is a whole number and compared as such
        return dict(logprobs=torch.cat(lp), entropy=torch.cat(ent), top_rows=None, top_logprobs=torch.cat(tops, 1))
    d, hk = case["dim"], case["h_kv"]
    if op == "window_attn":
        hq, n = case["h_q"], case["seq"]
        q, k, v = tensor(s["q"], hq * d), tensor(s["k"], hk * d), tensor(s["v"], hk * d)
        out = torch.empty(hq * d, s["cols"], dtype=torch.float64, device="cuda")
        t = torch.arange(n, device="cuda")
        age = t[:, None] - t[None, :]
        seen = age >= 0
        if case["window"]:
            seen &= (age < case["window"]) | (t < case["sinks"])[None, :]
        for f in range(case["frames"]):
            at = slice(f * n, (f + 1) * n)
            for h in range(hq):
                g = h // (hq // hk)
                qq, kk = _turn64(q[h * d: (h + 1) * d, at], t), _turn64(k[g * d: (g + 1) * d, at], t)
                out[h * d: (h + 1) * d, at] = _attend64(qq.t(), kk.t(), v[g * d: (g + 1) * d, at].t(), seen).t()
        return dict(out=out)
    cache = s["cache"]
    cols, nb = cache["codes"].shape[0], cache["codes"].shape[2]
    new = dict(codes=cache["codes"].double(), scales=cache["scales"].double(), k_tail=cache["k_tail"].double(), v_tail=cache["v_tail"].double(), tail_block=None)

    def keep(c, h, b, k, v):             # k, v [dim, 64] of one block; its unit is that of the FP16 numbers that the cache is given
        k = k.half().double()
        for which, x in ((0, k), (1, v)):
            unit = max(float(x.abs().max()), 2.0 ** -24) / 448.0
            new["scales"][c, h, b, which] = unit
            y = x / unit
            new["codes"][c, h, b, which] = torch.cat([y[i: i + 64].t().reshape(-1) for i in range(0, d, 64)]) if which == 0 else y.reshape(-1)

    if op == "kv8_fill":
        if case["frames"] * hk * (case["seq"] // 64 + 1) > 6000:
            return None
        k, v = tensor(s["k"], hk * d), tensor(s["v"], hk * d)
        n = case["seq"]
        for f, (slot, length) in enumerate(zip(s["slots"].tolist(), s["lengths"].tolist())):
            for h in range(hk):
                if length == 0:
                    continue
                at = slice(f * n, f * n + length)
                kk, vv = _turn64(k[h * d: (h + 1) * d, at], torch.arange(length, device="cuda")), v[h * d: (h + 1) * d, at]
                for b in range(length // 64):
                    keep(slot, h, b, kk[:, b * 64: b * 64 + 64], vv[:, b * 64: b * 64 + 64])
                r = length % 64
                if r:
                    new["k_tail"][slot, h, :r] = kk[:, -r:].t()
                    new["v_tail"][slot, h, :, :r] = vv[:, -r:]
        return new
    hq, g = case["h_q"], case["h_q"] // hk
    q, k, v = tensor(s["q"], hq * d), tensor(s["k"], hk * d), tensor(s["v"], hk * d)
    out = torch.zeros(hq * d, cols, dtype=torch.float64, device="cuda")
    for c, p in enumerate(s["pos"].tolist()):
        if p < 0:
            continue
        b, r = p // 64, p % 64
        at = torch.tensor([p], device="cuda")
        seen = torch.arange(p + 1, device="cuda")
        seen = torch.ones_like(seen, dtype=torch.bool) if case["window"] == 0 else (seen > p - case["window"]) | (seen < case["sinks"])
        for h in range(hk):
            new["k_tail"][c, h, r] = _turn64(k[h * d: (h + 1) * d, c: c + 1], at)[:, 0]
            new["v_tail"][c, h, :, r] = v[h * d: (h + 1) * d, c]
            kc = cache["codes"][c, h, :b, 0].double().reshape(b, d // 64, 64, 64) * cache["scales"][c, h, :b, 0].double()[:, None, None, None]
            vc = cache["codes"][c, h, :b, 1].double().reshape(b, d, 64) * cache["scales"][c, h, :b, 1].double()[:, None, None]
            kk = torch.cat([kc.permute(0, 2, 1, 3).reshape(b * 64, d), new["k_tail"][c, h, : r + 1]])
            vv = torch.cat([vc.permute(0, 2, 1).reshape(b * 64, d), new["v_tail"][c, h, :, : r + 1].t()])
            qq = _turn64(q[h * g * d: (h + 1) * g * d, c].view(g, d).t(), at.expand(g)).t()
            out[h * g * d: (h + 1) * g * d, c] = _attend64(qq, kk, vv, seen[None, :].expand(g, -1)).reshape(-1)
            if r == 63:
                keep(c, h, b, new["k_tail"][c, h].t(), new["v_tail"][c, h])
    return dict(out=out, **new)
