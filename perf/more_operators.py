"""What two additions around the paged cache are measured on: appending keys and values with the position rotation applied on the
way (queries too), and a cache held in 8 bits with one scale for each block of 16 tokens and kv head, with the attention that reads
it (single tokens, drafts, prompts).

A case is a dict of plain values:

  op                     "rotary"  rotate queries and keys by their positions, quantise keys and values into an NVFP4 cache
                         "append"  the same into the 8-bit cache, whose blocks may be part full already
                         "decode"  attention of a request's last tokens over the 8-bit cache
                         "prefill" attention of prompts, or chunks of prompts, over the 8-bit cache
  head_dim, kv_heads, group, page          the model's shape and the page size
  fmt                    codes of the 8-bit cache: "e4m3" or "int8"
  n, ctx_lo, ctx_hi      requests and their context lengths, log-uniform quantiles of [ctx_lo, ctx_hi] (append, prefill: cached
                         tokens before the new ones; rotary: tokens only, in slots at random)
  q_tokens               decode: query tokens of a request
  new_lo, new_hi         append, prefill: numbers of new tokens, log-uniform quantiles
  pad                    rotary, append: tokens at the end of the batch that have no slot (-1)
  rot, pairs, table      channels that are rotated (0: append without a rotation), which two belong together ("halves": i and
                         i + rot / 2, "neighbours": 2 i and 2 i + 1), type of the table of cosines and sines
  order, k8, had         rotary: the NVFP4 cache's page order, the slot with FP8 keys, keys multiplied by the Hadamard matrix
  window, sinks, lse     decode, prefill: visible keys (0: all), and whether the rows' log-sum-exps are wanted

The 8-bit cache. A tile is 16 tokens of one kv head and side: token t's row of D code bytes at t * D, its 16-byte chunk j at chunk
j ^ (t % 8), then the tile's scale, a power of two in fp32, and 12 unused bytes. value = code * scale * g with a global scale per kv
head. A write that names a tile's first token starts the tile anew, any other write keeps the tokens there: the scale is the larger of
the tile's own and the smallest power of two (of a range) with |code| <= 448 (e4m3) or 127 (int8), and where it grows, the codes that
are there are rounded to it.

Values: q, v ~ N(0, 1), k ~ N(0, 1) with four outlier channels per head scaled by 20. Outputs are the caches themselves: the NVFP4
cache and int8 codes as whole numbers, E4M3 codes as what they are, scales in fp32."""
import functools
import math
from types import SimpleNamespace

import torch

own = False

OUTLIER = 20.0
TABLE_ROWS = 131072
SHAPES = {"a": dict(head_dim=128, kv_heads=8, group=4), "b": dict(head_dim=128, kv_heads=8, group=8),
          "c": dict(head_dim=256, kv_heads=2, group=8), "d": dict(head_dim=256, kv_heads=4, group=6)}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
EXPONENTS = {"e4m3": (-15, 7), "int8": (-24, 9)}


def _case(name, op, shape, n, page=16, **more):
    c = dict(op=op, n=n, page=page, **SHAPES[shape])
    if op in ("rotary", "append"):
        c.update(rot=more.pop("rot", c["head_dim"]), pairs=more.pop("pairs", "halves"), table=more.pop("table", "fp32"), pad=more.pop("pad", 0))
    if op == "rotary":
        c.update(order=more.pop("order", "LBHNC"), k8=more.pop("k8", False), had=more.pop("had", False))
    else:
        c["fmt"] = more.pop("fmt", "e4m3")
        c["ctx_lo"], c["ctx_hi"] = more.pop("ctx")
    if op in ("append", "prefill"):
        c["new_lo"], c["new_hi"] = more.pop("new")
    if op in ("decode", "prefill"):
        c.update(window=more.pop("window", 0), sinks=more.pop("sinks", 0), lse=more.pop("lse", False))
    if op == "decode":
        c["q_tokens"] = more.pop("q", 1)
    c.update(more)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of each of a few users of a chat server, NVFP4 cache; the launch is most of it
        _case("rotary_four", "rotary", "a", 4),
        # a step of a batch at head_dim 256 whose model rotates a quarter of the channels, tokens up to a graph's size without a slot
        _case("rotary_step", "rotary", "d", 243, page=32, rot=64, table="bf16", pad=13),
        # the prompts of a step
        _case("rotary_fill", "rotary", "a", 16384),
        # one token each for a few users, 8-bit cache
        _case("append_four", "append", "a", 4, ctx=(1500, 6000), new=(1, 1)),
        # one token and a draft of another for every conversation of a busy server, int8 codes at head_dim 256
        _case("append_step", "append", "c", 256, page=32, fmt="int8", ctx=(500, 4096), new=(2, 2), pairs="neighbours"),
        # prompts of several lengths, some over a cached prefix that ends inside a block
        _case("append_fill", "append", "a", 12, ctx=(1, 3000), new=(300, 4000)),
        # a few users of one chat server
        _case("decode_four", "decode", "a", 4, ctx=(1500, 6000)),
        # a busy chat server
        _case("decode_batch", "decode", "a", 64, ctx=(1024, 32768)),
        # one draft token to verify at head_dim 256, int8 codes; the log-sum-exps join this with another part of the context
        _case("decode_verify", "decode", "c", 96, page=32, fmt="int8", ctx=(500, 16384), q=2, lse=True),
        # long documents
        _case("decode_long", "decode", "b", 8, ctx=(65536, 65536)),
        # a fresh prompt
        _case("prefill_prompt", "prefill", "a", 1, ctx=(0, 0), new=(4096, 4096)),
        # a chunk of a long prompt over its cached part, int8 codes at head_dim 256
        _case("prefill_chunk", "prefill", "c", 1, fmt="int8", ctx=(16000, 16000), new=(2048, 2048), lse=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "decode", "prefill"))
    shape = rng.choice(("a", "a", "b", "c", "d"))
    page = rng.choice((16, 16, 32, 64))
    D, H = SHAPES[shape]["head_dim"], SHAPES[shape]["kv_heads"]
    fmt = rng.choice(("e4m3", "e4m3", "int8"))
    if op in ("rotary", "append"):
        turn = dict(rot=rng.choice((D, D, D, 64, 48, 16 * rng.randint(1, D // 16))), pairs=rng.choice(("halves", "halves", "neighbours")),
                    table=rng.choice(("fp32", "bf16")), pad=rng.choice((0, 0, rng.randint(1, 40))))
    if op == "rotary":
        opt = rng.choice(({}, {}, {}, {"order": "LBNHC"}, {"k8": True}, {"had": True}))
        if "k8" in opt and D != 256:
            opt = {}
        return _case(None, op, shape, _log(rng, 1, 16384 * 1024 // (H * D)), page, **turn, **opt)
    if op == "append":
        if rng.random() < 0.2:
            turn["rot"] = 0
        if rng.random() < 0.5:
            new = rng.choice((1, 1, 1, 2, 4))
            return _case(None, op, shape, _log(rng, 1, 512), page, fmt=fmt, ctx=(_log(rng, 1, 500), _log(rng, 500, 4096)), new=(new, new), **turn)
        n = rng.choice((1, 2, 5, 12))
        new = _log(rng, 3, 16384 * 1024 // (H * D) // n)
        prior = 0 if rng.random() < 0.4 else _log(rng, 1, 3000)
        return _case(None, op, shape, n, page, fmt=fmt, ctx=(prior // 2, prior), new=(max(1, new // 8), new), **turn)
    window = 0 if rng.random() < 0.7 else _log(rng, 1, 8192)
    see = dict(window=window, sinks=rng.choice((0, 4, 20)) if window else 0, lse=rng.random() < 0.3)
    if op == "decode":
        hi = _log(rng, 48, 65536)
        n = _log(rng, 1, max(1, min(256, 2 ** 29 // (H * D) // hi)))
        return _case(None, op, shape, n, page, fmt=fmt, ctx=(_log(rng, max(1, hi // 64), hi), hi), q=rng.choice((1, 1, 1, 2, 4)), **see)
    n = rng.choice((1, 1, 2, 4))
    new = _log(rng, 9, 4096 // n)
    prior = 0 if rng.random() < 0.5 else _log(rng, 64, 16000)
    while n * new * (prior + new) * H * SHAPES[shape]["group"] * D > 2048 * 18048 * 16 * 256:
        prior, new = prior * 2 // 3, max(9, new * 3 // 4)
    return _case(None, op, shape, n, page, fmt=fmt, ctx=(prior // 2, prior), new=(max(4, new // 2), new), **see)


# ------------------------------------------------------------------------------------------------------------ lengths
def _quantiles(n, lo, hi):
    """n values of a log-uniform law on [lo, hi] (lo = 0 counts as 1, less one), by their quantiles"""
    off = 1 if lo == 0 else 0
    a, b = math.log(lo + off), math.log(hi + off)
    return [int(round(math.exp(a + (b - a) * (i + 0.5) / n))) - off for i in range(n)]


def _requests(case):
    """[(new or query tokens, context length with them)]"""
    ctx = _quantiles(case["n"], case["ctx_lo"], case["ctx_hi"])
    if case["op"] == "decode":
        return [(case["q_tokens"], max(case["q_tokens"], L)) for L in ctx]
    return [(q, q + p) for q, p in zip(_quantiles(case["n"], case["new_lo"], case["new_hi"]), reversed(ctx))]


def _tokens(case):
    return case["n"] if case["op"] == "rotary" else sum(q for q, _ in _requests(case))


# ------------------------------------------------------------------------------------------------------------ prepare
def _keys(g, *shape):
    k = torch.randn(*shape, generator=g, device="cuda")
    D = shape[-1]
    k[..., [3, D // 4 + 3, D // 2 + 3, 3 * D // 4 + 3]] *= OUTLIER
    return k


def _table(case):
    """cosines, then sines, of every position: rows of `rot` numbers"""
    half = case["rot"] // 2
    step = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    a = torch.arange(TABLE_ROWS, dtype=torch.float64, device="cuda")[:, None] * step
    return torch.cat((a.cos(), a.sin()), 1).to(torch.bfloat16 if case["table"] == "bf16" else torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 6151 + 71)
    H, D, G, PS = case["kv_heads"], case["head_dim"], case["group"], case["page"]
    s = SimpleNamespace(op=case["op"], H=H, D=D, G=G, page=PS, ws=None)
    if case["op"] in ("rotary", "append"):
        s.rot, s.neighbours, n = case["rot"], case["pairs"] == "neighbours", _tokens(case)
        # queries, keys and values as one product of a layer leaves them, side by side
        HQ = H * G
        qkv = torch.randn(n + case["pad"], (HQ + 2 * H) * D, generator=g, device="cuda")
        qkv[:, HQ * D:(HQ + H) * D] = _keys(g, n + case["pad"], H, D).flatten(1)
        qkv = qkv.to(torch.bfloat16)
        s.q, s.k, s.v = (x.view(-1, h, D) for x, h in zip(qkv.split((HQ * D, H * D, H * D), 1), (HQ, H, H)))
        s.q_out = torch.zeros((n + case["pad"], HQ, D), dtype=torch.bfloat16, device="cuda")
        s.table = _table(case) if s.rot else None
    if case["op"] == "rotary":
        return _prepare_rotary(s, case, g)
    s.fmt = case["fmt"]
    reqs = _requests(case)
    mix = torch.randperm(len(reqs), generator=torch.Generator().manual_seed(seed + 3)).tolist()
    reqs = [reqs[i] for i in mix]
    B, T = len(reqs), sum(q for q, _ in reqs)
    pages = torch.tensor([(L + PS - 1) // PS for _, L in reqs])
    MP, total = int(pages.max()), int(pages.sum())
    pool = (torch.randperm(total, generator=g, device="cuda") + 1).to(torch.int32)
    bt = torch.zeros((B, MP), dtype=torch.int32, device="cuda")
    bt[(torch.arange(MP) < pages[:, None]).cuda()] = pool
    phys = torch.zeros((total + 1, 2 * H, PS // 16, 16 * D + 16), dtype=torch.uint8, device="cuda")
    s.tiles, s.bt = phys, bt
    s.flat = (phys.view(-1), phys.view(-1)[H * phys.stride(1):])
    s.strides = (phys.stride(0), phys.stride(1))
    s.swap = _swap(D)
    # (the global scales are what a server calibrates: a round number near the largest value)
    s.gk = torch.full((H,), 1.0, device="cuda")
    s.gv = torch.full((H,), 1.0, device="cuda")
    s.lens = torch.tensor([L for _, L in reqs], dtype=torch.int32, device="cuda")
    s.qlens = [q for q, _ in reqs]
    s.qsl = torch.tensor([0] + s.qlens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    s.row_of = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(s.qlens, device="cuda"))
    s.tok_of = torch.arange(T, device="cuda") - s.qsl[s.row_of].long()
    s.q_len = torch.tensor(s.qlens, device="cuda")
    _fill(s, g)
    if case["op"] == "append":
        pos = (s.lens - s.q_len)[s.row_of].long() + s.tok_of
        page = s.bt.long()[s.row_of, pos // PS]
        off = torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")
        s.slots = torch.cat((page * PS + pos % PS, off))
        s.positions = torch.cat((pos, torch.zeros_like(off)))
        # the tiles that the step writes to, and which of them a token belongs to
        s.touched, s.tile_of = torch.unique(s.slots[:T] // 16, return_inverse=True)
        return s
    s.B, s.qlmax, s.sm = B, max(s.qlens), D ** -0.5
    s.window, s.sinks = case["window"], case["sinks"]
    s.q = torch.randn(T, H * G, D, generator=g, device="cuda").to(torch.bfloat16)
    s.out = torch.zeros_like(s.q)
    s.lse = torch.zeros(T, H * G, device="cuda") if case["lse"] else None
    s.rows = [(b, a, a + q, L) for b, (a, (q, L)) in enumerate(zip(s.qsl.tolist(), reqs))]
    s.reach = max(L for _, L in reqs)
    return s


def _prepare_rotary(s, case, g):
    H, D, PS, n = s.H, s.D, s.page, case["n"]
    s.k8, s.had = case["k8"], case["had"]
    slot = D + D // 2 + D // 16 if s.k8 else D // 2 + D // 16
    heads, pages = (H if s.k8 else 2 * H), (n + PS - 1) // PS + 1
    if case["order"] == "LBNHC":
        phys = torch.zeros((pages, PS, heads, slot), dtype=torch.uint8, device="cuda")
        s.cache = phys.permute(0, 2, 1, 3)
    else:
        phys = s.cache = torch.zeros((pages, heads, PS, slot), dtype=torch.uint8, device="cuda")
    s.phys = phys
    parts = (0, D, D, D + D // 2) if s.k8 else (0, D // 2, H * s.cache.stride(1), H * s.cache.stride(1) + D // 2)
    st = (s.cache.stride(0), s.cache.stride(2), s.cache.stride(1))
    s.flat, s.strides = tuple(phys.view(-1)[p:] for p in parts), st + st
    off = torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")
    s.slots = torch.cat((torch.randperm(pages * PS, generator=g, device="cuda")[:n], off))
    s.positions = torch.randint(0, TABLE_ROWS, (n + case["pad"],), generator=g, device="cuda")
    s.gk = torch.full((H,), OUTLIER * 5.5 / (448 if s.k8 else 6 * 448), device="cuda")
    s.gv = torch.full((H,), 5.5 / (6 * 448), device="cuda")
    s.signs = None
    if s.had:
        s.signs = (torch.randint(0, 2, (D,), generator=torch.Generator().manual_seed(0x6B7634)) * 2 - 1).float().cuda()
    return s


def _fill(s, g):
    """keys and values of all pages, as the cache's writer leaves full tiles"""
    n = s.tiles.shape[0]
    step = max(1, 2 ** 26 // (s.H * s.page * s.D))
    for i in range(0, n, step):
        m = min(step, n - i)
        shape = (m, s.H, s.page // 16, 16, s.D)
        x = torch.cat((_keys(g, *shape), torch.randn(*shape, generator=g, device="cuda")), 1).to(torch.bfloat16).float()
        scale = _scale(x.abs().amax((-1, -2)), s.fmt)
        code = _bytes(x / scale[..., None, None], s.fmt).gather(-1, s.swap.expand(x.shape))
        s.tiles[i:i + m, :, :, :16 * s.D] = code.flatten(-2)
        s.tiles[i:i + m, :, :, 16 * s.D:16 * s.D + 4] = scale[..., None].view(torch.uint8)


# --------------------------------------------------------------------------------------------------------- plain forms
def _rotate(s, x):
    """x (T, heads, D) bf16, each position's pairs turned by its angles, rounded once to bf16"""
    if not s.rot:
        return x
    c, sn = s.table.index_select(0, s.positions).float()[:, None].chunk(2, -1)
    y = x.float()
    a, b = (y[..., 0:s.rot:2], y[..., 1:s.rot:2]) if s.neighbours else y[..., :s.rot].chunk(2, -1)
    a, b = a * c - b * sn, b * c + a * sn
    turned = torch.stack((a, b), -1).flatten(-2) if s.neighbours else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., s.rot:]), -1).to(torch.bfloat16)


def _stage(y, h):
    v = y.unflatten(-1, (-1, 2, h))
    return torch.stack((v[..., 0, :] + v[..., 1, :], v[..., 0, :] - v[..., 1, :]), -2).flatten(-3)


def _e4m3_byte(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _fp4(x, g):
    """(T, H, D) fp32 and the heads' global scales -> (T, H, D / 2 + D / 16) bytes: E2M1 codes two to a byte, then the block scales.
    A block's scale is the one of four with the least squared error, the first of them among equals."""
    b = x.unflatten(-1, (-1, 16))
    mag, g = b.abs(), g[:, None]
    amax = mag.amax(-1)
    near, far = _e4m3_byte(amax / (g * 6.0)).int(), _e4m3_byte(amax / (g * 4.0)).int()
    byte = torch.stack((near, (near + 1).clamp(max=126), (near - 1).clamp(min=0), far), -1).to(torch.uint8)
    scale = (byte.view(torch.float8_e4m3fn).float() * g[..., None])[..., None]
    y = torch.where(scale > 0, mag[..., None, :] / scale, 0.0)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    value = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0), device=x.device)[code.int()]
    d = value * scale - mag[..., None, :]
    err = functools.reduce(torch.add, (d * d).unbind(-1))              # (in the order of the channels)
    best = torch.where(err == err.amin(-1, keepdim=True), torch.arange(4, device=x.device), 4).amin(-1, keepdim=True)
    code = code.gather(-2, best[..., None].expand(*best.shape, 16))[..., 0, :] | (b < 0).to(torch.uint8) << 3
    code = code.unflatten(-1, (-1, 2))
    return torch.cat(((code[..., 0] | code[..., 1] << 4).flatten(-2), byte.gather(-1, best)[..., 0]), -1)


def _plain_rotary(s):
    s.q_out.copy_(_rotate(s, s.q))
    on = s.slots >= 0
    k, v = _rotate(s, s.k)[on].float(), s.v[on].float()
    if s.had:
        stages = [2 ** i for i in range(s.D.bit_length() - 1)]
        k = functools.reduce(_stage, stages, k * s.signs) * float(torch.tensor(s.D ** -0.5, dtype=torch.float32))
    k = _e4m3_byte(k / s.gk[:, None]) if s.k8 else _fp4(k, s.gk)
    v = _fp4(v, s.gv)
    page, pos = s.slots[on] // s.page, s.slots[on] % s.page
    s.cache[page, :, pos] = torch.cat((k, v), 2 if s.k8 else 1)


def _swap(D):
    """where channel c of token t lies in its row: (16, D)"""
    t, c = torch.arange(16, device="cuda")[:, None], torch.arange(D, device="cuda")
    return (c // 16 ^ t % 8) * 16 + c % 16


def _scale(amax, fmt):
    """the smallest power of two with amax / scale within the codes, of the exponents that there are"""
    m, e = torch.frexp(amax)                                           # amax = m 2^e, 0.5 <= m < 1
    top_m, top_e = math.frexp(LARGEST[fmt])
    e = torch.where(amax > 0, e - top_e + (m > top_m).int(), EXPONENTS[fmt][0]).clamp(*EXPONENTS[fmt])
    return (e + 127 << 23).view(torch.float32)


def _bytes(y, fmt):
    return _e4m3_byte(y) if fmt == "e4m3" else y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)


def _codes(b, fmt):
    return b.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float()


def _plain_append(s):
    D, n = s.D, s.tile_of.numel()
    if s.rot:
        s.q_out.copy_(_rotate(s, s.q))
    x = torch.cat((_rotate(s, s.k)[:n].float() / s.gk[:, None], s.v[:n].float() / s.gv[:, None]), 1)       # (n, 2 H, D)
    per = s.page // 16
    page, sub, at = s.touched // per, s.touched % per, s.slots[:n] % 16
    old = s.tiles[page, :, sub]                                        # (tiles, 2 H, 16 D + 16)
    had = old[..., 16 * D:16 * D + 4].contiguous().view(torch.float32)
    new = torch.zeros(old.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, s.tile_of[at == 0], True)[:, None, None]
    amax = torch.zeros(old.shape[:2], device="cuda").scatter_reduce_(0, s.tile_of[:, None].expand(x.shape[:2]), x.abs().amax(-1), "amax")
    scale = _scale(amax, s.fmt)[..., None]
    scale = torch.where(new, scale, torch.maximum(scale, had))
    swap = s.swap.expand(*old.shape[:2], 16, D)
    code = old[..., :16 * D].unflatten(-1, (16, D))
    code = torch.where((new | (scale == had))[..., None], code, _bytes(_codes(code.contiguous(), s.fmt) * (had / scale)[..., None], s.fmt))
    code = code.gather(-1, swap)                                       # rows in the order of their channels
    code[s.tile_of, :, at] = _bytes(x / scale[s.tile_of], s.fmt)
    s.tiles[page, :, sub] = torch.cat((code.gather(-1, swap).flatten(-2), scale.view(torch.uint8), old[..., 16 * D + 4:]), -1)


def _plain_attention(s):
    """(B, H, N) keys and values side by side, padded to the longest context"""
    dev, L = "cuda", s.lens.long()
    pos = torch.arange(s.reach, device=dev)
    at = pos.minimum(L[:, None] - 1)
    page, row = torch.gather(s.bt.long(), 1, at // s.page), at % s.page
    tile = s.tiles.view(-1, 2 * s.H, s.page // 16, 16 * s.D + 16)
    code = tile[..., :16 * s.D].unflatten(-1, (16, s.D))[page, :, row // 16, row % 16]                    # (B, N, 2 H, D)
    scale = tile[..., 16 * s.D:16 * s.D + 4].contiguous().view(torch.float32)[page, :, row // 16]           # (B, N, 2 H, 1)
    code = code.gather(-1, s.swap[row % 16][:, :, None].expand(code.shape))
    k, v = (_codes(code, s.fmt) * scale).permute(0, 2, 1, 3).chunk(2, 1)
    del code
    qp = torch.zeros(s.B, s.H, s.qlmax, s.G, s.D, device=dev)
    qp[s.row_of, :, s.tok_of] = s.q.float().view(-1, s.H, s.G, s.D)
    x = qp.view(s.B, s.H, s.qlmax * s.G, s.D) @ (k * (s.sm * s.gk[:, None, None])).transpose(2, 3)
    del k
    p = (L - s.q_len)[:, None] + torch.arange(s.qlmax, device=dev)         # positions of the query tokens
    see = pos <= p[..., None]
    if s.window:
        see &= (pos > p[..., None] - s.window) | (pos < s.sinks)
    see &= (torch.arange(s.qlmax, device=dev) < s.q_len[:, None])[..., None]
    x = torch.where(see[:, None, :, None].expand(-1, s.H, -1, s.G, -1).reshape(x.shape), x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = (x - m).exp()
    del x
    den = e.sum(-1, keepdim=True)
    o = e @ v / torch.where(den > 0, den, 1.0) * s.gv[:, None, None]
    shape = (s.B, s.H, s.qlmax, s.G)
    s.out.copy_(o.view(*shape, s.D)[s.row_of, :, s.tok_of].reshape(s.out.shape))
    if s.lse is not None:
        s.lse.copy_((m + den.log()).view(shape)[s.row_of, :, s.tok_of].reshape(s.lse.shape))


_K = None


def _kernels():
    global _K
    if _K is None:
        from horizon_kernels_b200 import kernels
        _K = kernels
    return _K


def _workspace(s):
    if s.ws is None:                              # made once, as a program keeps it
        s.ws = _kernels().alloc_workspace(s.B, s.H, s.G, s.D, s.qlmax if s.op == "decode" else 1)
    return s.ws


def _cache8(s):
    """the 8-bit cache as what its bytes stand for: codes and scales"""
    code = s.tiles[..., :16 * s.D].view(torch.float8_e4m3fn if s.fmt == "e4m3" else torch.int8)
    return {"codes": code, "scales": s.tiles[..., 16 * s.D:16 * s.D + 4].view(torch.float32)}


def run(state):
    s = state
    if s.op == "rotary":
        if own:
            _kernels().write_rotary(s.q, s.k, s.v, s.flat, s.strides, s.page, s.slots, s.positions, s.table, s.gk, s.gv, s.q_out,
                                    interleaved=s.neighbours, signs=s.signs, k8=s.k8)
        else:
            _plain_rotary(s)
        return {"query": s.q_out, "cache": s.phys}
    if s.op == "append":
        if not own:
            _plain_append(s)
        elif s.rot:
            _kernels().write_rotary_b8(s.q, s.k, s.v, s.flat, s.strides, s.page, s.slots, s.positions, s.table, s.gk, s.gv, s.q_out,
                                       interleaved=s.neighbours, fmt=s.fmt)
        else:
            _kernels().write_b8(s.k, s.v, s.flat, s.strides, s.page, s.slots, s.gk, s.gv, fmt=s.fmt)
        return {"query": s.q_out if s.rot else None, **_cache8(s)}
    if not own:
        _plain_attention(s)
    elif s.op == "decode":
        _kernels().decode_b8(s.q, s.flat, s.strides, s.page, s.bt, s.lens, s.qsl, s.sm, 1.0, s.gk, s.gv, s.qlmax, s.out,
                             _workspace(s), fmt=s.fmt, window=s.window, sinks=s.sinks, lse=s.lse)
    else:
        _kernels().prefill_b8(s.q, s.flat, s.strides, s.page, s.bt, s.rows, s.sm, 1.0, s.H, s.out, fmt=s.fmt, window=s.window,
                              sinks=s.sinks, workspace=_workspace(s), lse=s.lse)
    return {"out": s.out, "lse": s.lse}


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    H, D, PS = case["kv_heads"], case["head_dim"], case["page"]
    HQ = H * case["group"]
    if case["op"] in ("rotary", "append"):
        T = _tokens(case)
        turned = (HQ + H) * case["rot"]                                # channels of a token
        n = T * (2 * H * D * 2 + 8) + 8 * H
        if case["rot"]:
            n += (T + case["pad"]) * (2 * HQ * D * 2 + 8 + case["rot"] * (2 if case["table"] == "bf16" else 4))
        if case["op"] == "rotary":
            n += T * H * (D + D // 2 + D // 16 if case["k8"] else 2 * (D // 2 + D // 16))
        else:
            n += T * 2 * H * D
            for q, L in _requests(case):                               # tiles' scales: read where a tile is part full, written
                n += 2 * H * 4 * ((L + 15) // 16 - (L - q) // 16 + ((L - q) % 16 > 0))
        return {"bytes": n, "flops": 3 * T * turned}
    n = flops = 0
    for q, L in _requests(case):
        lo = max(0, L - q - case["window"] + 1) if case["window"] else 0
        seen = L - lo + min(lo, case["sinks"])                         # tokens that some row sees
        n += seen * H * 2 * D + (seen + 15) // 16 * H * 2 * 4 + 4 * (seen + PS - 1) // PS + 12 + q * HQ * (4 * D + 4 * case["lse"])
        flops += 4 * D * HQ * sum(_pairs(case, L - q + t) for t in range(q))
    return {"bytes": n, "flops": flops}


def _pairs(case, p):
    """keys that the query token at position p sees"""
    lo = max(0, p - case["window"] + 1) if case["window"] else 0
    return p + 1 - lo + min(lo, case["sinks"])


# --------------------------------------------------------------------------------------------------------------- exact
def _turned64(s, x):
    """x in 64 bits, every pair of channels as a complex number times e^(i angle)"""
    y = x.double()
    if not s.rot:
        return y
    half = s.rot // 2
    row = s.table[s.positions].double()
    at = torch.arange(half, device="cuda")
    a, b = (2 * at, 2 * at + 1) if s.neighbours else (at, at + half)
    z = torch.complex(y[..., a], y[..., b]) * torch.complex(row[:, :half], row[:, half:])[:, None]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_append(s):
    D = s.D
    query = _turned64(s, s.q) if s.rot else None
    tiles, T = s.tiles, s.tile_of.numel()
    bits = tiles[..., :16 * D].view(torch.float8_e4m3fn if s.fmt == "e4m3" else torch.int8).double().view(*tiles.shape[:3], 16, D // 16, 16)
    t, j = torch.arange(16, device="cuda")[:, None], torch.arange(D // 16, device="cuda")
    code = bits[:, :, :, t, j ^ (t & 7)]                               # chunks in order
    scale = tiles[..., 16 * D:16 * D + 4].contiguous().view(torch.float32).double()[..., 0]
    k = _turned64(s, s.k).to(torch.bfloat16).double() / s.gk.double()[:, None]
    x = torch.cat((k, s.v.double() / s.gv.double()[:, None]), 1)[:T]
    per, lo, hi = s.page // 16, *EXPONENTS[s.fmt]
    page, sub = s.touched // per, s.touched % per
    big = torch.zeros((s.touched.numel(), 2 * s.H), dtype=torch.float64, device="cuda")
    big.scatter_reduce_(0, s.tile_of[:, None].expand(-1, 2 * s.H), x.abs().amax(-1), "amax")
    m, e = torch.frexp((big / LARGEST[s.fmt]).clamp(min=2.0 ** lo, max=2.0 ** hi))
    need = _two64(torch.where(m == 0.5, e - 1, e))
    start = torch.isin(torch.arange(s.touched.numel(), device="cuda"), s.tile_of[s.slots[:T] % 16 == 0])
    was, vals = scale[page, :, sub], code[page, :, sub]
    now = torch.where(start[:, None], need, torch.maximum(need, was))
    grown = ~start[:, None] & (now > was)
    vals = torch.where(grown[..., None, None, None], _nearest64(vals * (was / now)[..., None, None, None], s.fmt), vals)
    vals[s.tile_of, :, s.slots[:T] % 16] = _nearest64(x / now[s.tile_of][..., None], s.fmt).unflatten(-1, (-1, 16))
    code[page, :, sub], scale[page, :, sub] = vals, now
    if s.fmt == "int8":
        return {"query": query, "codes": None, "scales": scale[..., None]}
    return {"query": query, "codes": code[:, :, :, t, j ^ (t & 7)].flatten(-3), "scales": scale[..., None]}


def _two64(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _nearest64(y, fmt):
    """the nearest code, ties to the even one, in 64 bits"""
    if fmt == "int8":
        return y.round().clamp(-127, 127)
    step = _two64(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)   # three mantissa bits, subnormals in steps of 2^-9
    return ((y / step).round() * step).clamp(-448, 448)


def _values64(s, b, L, h, side):
    pos = torch.arange(L, device="cuda")
    page = s.bt[b, pos // s.page].long()
    tile = s.tiles[page, h + side * s.H, pos % s.page // 16]           # (L, 16 D + 16)
    chunk = torch.arange(s.D // 16, device="cuda") ^ (pos % 8)[:, None]
    at = ((pos % 16 * s.D)[:, None] + chunk * 16)[..., None] + torch.arange(16, device="cuda")
    code = tile.gather(1, at.flatten(1)).view(torch.float8_e4m3fn if s.fmt == "e4m3" else torch.int8).double()
    return code * tile[:, 16 * s.D:16 * s.D + 4].contiguous().view(torch.float32).double()


def exact(case, seed):
    """Every operator from its definition in 64 bits: rotations as complex products, codes by rounding, attention head by head. Whole
    numbers (the NVFP4 cache, int8 codes) have no value here."""
    s = prepare(case, seed)
    if s.op == "rotary":
        return {"query": _turned64(s, s.q), "cache": None}
    if s.op == "append":
        return _exact_append(s)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s.q.shape[:2], dtype=torch.float64, device="cuda")
    for b, a, e, L in s.rows:
        pos, place = torch.arange(L, device="cuda"), torch.arange(L - (e - a), L, device="cuda")
        for h in range(s.H):
            k, v = _values64(s, b, L, h, 0), _values64(s, b, L, h, 1)
            heads = slice(h * s.G, (h + 1) * s.G)
            step = max(1, 2 ** 28 // (s.G * L))                        # (query tokens at a time)
            for i in range(0, e - a, step):
                p = place[i:i + step, None]
                see = pos <= p
                if s.window:
                    see &= (p - pos < s.window) | (pos < s.sinks)
                rows = slice(a + i, min(a + i + step, e))
                x = s.q[rows, heads].double() @ k.T * (s.sm * s.gk[h].double())
                x = x.masked_fill(~see[:, None], -math.inf)
                l = torch.logsumexp(x, -1)
                out[rows, heads] = (x - l[..., None]).exp() @ v * s.gv[h].double()
                lse[rows, heads] = l
    return {"out": out, "lse": lse if s.lse is not None else None}
