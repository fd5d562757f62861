"""What the operators for bounded caches are measured on: attention over a sliding window and the first tokens (decode and
prefill rows), the attention weight that cached tokens have gathered, and the eviction that goes by it. All of them work on
a paged NVFP4 cache: E2M1 codes with an E4M3 scale per 16 channels, head-major or positions-outermost pages, or the slot
with FP8 keys.

A case is a dict of plain values:

  op                      "decode", "prefill", "weights" or "evict"
  head_dim, kv_heads, group, page, order, k8, had   the model's shape and the cache's options (had: rotated keys)
  n, ctx_lo, ctx_hi       requests and their context lengths, log-uniform quantiles of [ctx_lo, ctx_hi] (prefill: cached tokens
                          before the new ones)
  q_tokens                query tokens of a decode request, or the tokens whose attention is observed
  new_lo, new_hi          prefill: numbers of new tokens, log-uniform quantiles
  window, sinks           a query token at position p sees the keys p - window + 1 .. p and those below sinks (window 0: all)
  lse                     the log-sum-exp of the rows is wanted too
  keep, recent            evict: tokens that stay, and how many of the last ones among them (the first `sinks` too)

Values: q and v ~ N(0, 1), k ~ N(0, 1) with four outlier channels per head scaled by 20, quantised block by block; global
scales amax / (6 * 448) (FP8 keys: amax / 448); pages scattered at random over the pool. Pages that no row sees are not in
the pool: their table entries name page 0, which holds NaN scales, as an engine leaves them that frees what falls out of the
window. Weights to evict by are log-normal with a tenth of them zero, those to add to are small. The lengths follow from the case alone."""
import math
from types import SimpleNamespace

import torch

own = False

OUTLIER = 20.0
SHAPES = {"a": dict(head_dim=128, kv_heads=8, group=4), "b": dict(head_dim=128, kv_heads=8, group=8),
          "c": dict(head_dim=256, kv_heads=2, group=8), "d": dict(head_dim=256, kv_heads=4, group=6)}


def _case(name, op, shape, n, ctx, page=16, order="LBHNC", k8=False, had=False, **more):
    c = dict(op=op, n=n, ctx_lo=ctx[0], ctx_hi=ctx[1], page=page, order=order, k8=k8, had=had, **SHAPES[shape])
    if op != "evict":
        c.update(q_tokens=more.pop("q", 1), window=more.pop("window", 0), sinks=more.pop("sinks", 0), lse=more.pop("lse", False))
    if op == "prefill":
        c["new_lo"], c["new_hi"] = more.pop("new")
    c.update(more)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few users of one chat server whose conversations have grown past the window; launches are most of it
        _case("window_four", "decode", "a", 4, (1500, 6000), window=1024, sinks=4),
        # a busy chat server that bounds every conversation to 4096 tokens, contexts up to 131072; the rows' log-sum-exps feed
        # the gathered weights
        _case("window_batch", "decode", "a", 64, (1024, 131072), window=4096, sinks=4, lse=True),
        # one draft token to verify at head_dim 256, a window that is no multiple of anything
        _case("window_verify", "decode", "c", 96, (500, 16384), q=2, window=2047, sinks=5, page=32),
        # a fresh prompt, much longer than the window
        _case("window_prompt", "prefill", "a", 1, (0, 0), new=(6144, 6144), window=1024, sinks=4),
        # a chunk of a long prompt over its cached part, at head_dim 256
        _case("window_chunk", "prefill", "c", 1, (30000, 30000), new=(2048, 2048), window=4096, sinks=16, lse=True),
        # prompts of several lengths, some with a cached prefix, that start in one step
        _case("window_prompts", "prefill", "b", 4, (1, 3000), new=(90, 1500), window=500, sinks=3),
        # the weights of a small decode step
        _case("weights_four", "weights", "a", 4, (2048, 2048)),
        # the same over long documents
        _case("weights_long", "weights", "b", 8, (131072, 131072)),
        # the last four tokens of each prompt vote on what of it stays, at head_dim 256 (32 query rows per kv head)
        _case("weights_observe", "weights", "c", 32, (1000, 16384), q=4),
        # one conversation is cut from 8192 to 2048 tokens
        _case("evict_one", "evict", "a", 1, (8192, 8192), keep=2048, sinks=4, recent=256),
        # a batch of conversations of different lengths, some of which still fit
        _case("evict_batch", "evict", "a", 64, (1500, 16384), keep=2048, sinks=4, recent=512, page=32),
        # long documents at head_dim 256, positions-outermost pages
        _case("evict_long", "evict", "c", 8, (131072, 131072), keep=16384, sinks=16, recent=1024, order="LBNHC"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("decode", "prefill", "weights", "evict"))
    shape = rng.choice(("a", "a", "b", "c", "d"))
    opt = rng.choice(({}, {}, {}, {"order": "LBNHC"}, {"k8": True}, {"had": True}))
    if "k8" in opt and SHAPES[shape]["head_dim"] != 256:
        shape = rng.choice(("c", "d"))
    row = SHAPES[shape]["kv_heads"] * SHAPES[shape]["head_dim"]         # values of one token and side
    page = rng.choice((16, 16, 32, 64))
    window = _log(rng, 1, 8192)
    sinks = rng.choice((0, 1, 4, 16, 100))
    if op == "decode":
        hi = _log(rng, 64, 131072)
        seen = min(hi, window + sinks)
        n = _log(rng, 1, max(1, min(256, 2 ** 28 // row // seen)))       # up to 2^28 visible values per side
        return _case(None, op, shape, n, (_log(rng, max(1, hi // 64), hi), hi), page, q=rng.choice((1, 1, 1, 2, 4)), window=window,
                     sinks=sinks, lse="had" not in opt and rng.random() < 0.5, **opt)
    if op == "prefill":
        n = rng.choice((1, 1, 2, 4))
        new = _log(rng, 16, 6144 // n)
        prior = 0 if rng.random() < 0.5 else _log(rng, 64, 30000)
        window = _log(rng, 16, 4096)
        while n * new * (min(prior, window) + window + new) * SHAPES[shape]["group"] * row > 2048 * 6000 * 8 * 512:
            new = max(16, new * 2 // 3)
            window = max(16, window * 3 // 4)
        return _case(None, op, shape, n, (prior // 2, prior), page, new=(max(4, new // 2), new), window=window, sinks=sinks,
                     lse="had" not in opt and rng.random() < 0.3, **opt)
    if op == "weights":
        opt.pop("had", None)
        hi = _log(rng, 64, 131072)
        n = _log(rng, 1, max(1, min(256, 2 ** 28 // row // hi)))
        if rng.random() < 0.7:
            window = sinks = 0
        return _case(None, op, shape, n, (_log(rng, max(1, hi // 64), hi), hi), page, q=rng.choice((1, 1, 1, 2, 4)), window=window,
                     sinks=sinks, **opt)
    opt.pop("had", None)
    hi = _log(rng, 64, 131072)
    keep = _log(rng, 16, max(16, hi))
    n = _log(rng, 1, max(1, min(256, 2 ** 28 // row // hi)))
    sinks = min(sinks, keep // 4)
    return _case(None, op, shape, n, (_log(rng, max(1, hi // 16), hi), hi), page, keep=keep, sinks=sinks,
                 recent=rng.randint(0, keep - sinks), **opt)


# ------------------------------------------------------------------------------------------------------------ lengths
def _quantiles(n, lo, hi):
    """n values of a log-uniform law on [lo, hi] (lo = 0 counts as 1, less one), by their quantiles"""
    off = 1 if lo == 0 else 0
    a, b = math.log(lo + off), math.log(hi + off)
    return [int(round(math.exp(a + (b - a) * (i + 0.5) / n))) - off for i in range(n)]


def _requests(case):
    """[(query tokens, context length with them)]"""
    ctx = _quantiles(case["n"], case["ctx_lo"], case["ctx_hi"])
    if case["op"] == "prefill":
        return [(q, q + p) for q, p in zip(_quantiles(case["n"], case["new_lo"], case["new_hi"]), reversed(ctx))]
    q = case.get("q_tokens", 1)
    return [(q, max(q, L)) for L in ctx]


def _first_seen(case, q, L):
    """first position of the window of a request's first query token (0: everything is seen)"""
    return max(0, L - q - case["window"] + 1) if case.get("window") else 0


def _seen(case, q, L):
    """tokens that some query row of the request sees"""
    lo = _first_seen(case, q, L)
    return L - lo + min(lo, case.get("sinks", 0))


# ------------------------------------------------------------------------------------------------------------ prepare
_EDGES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _quantise(x, scale):
    """(.., D) fp32 -> (.., D / 2 + D / 16) bytes: codes two to a byte, then the block scales"""
    b = x.reshape(*x.shape[:-1], -1, 16) / scale
    sf = (b.abs().amax(-1) / 6).to(torch.float8_e4m3fn)
    y = b / sf.float().clamp_min(2.0 ** -9)[..., None]
    code = torch.bucketize(y.abs(), torch.tensor(_EDGES, device=x.device)).to(torch.uint8) | (y < 0).to(torch.uint8) << 3
    code = code.reshape(*x.shape[:-1], -1, 2)
    return torch.cat((code[..., 0] | code[..., 1] << 4, sf.view(torch.uint8)), dim=-1)


def _fill(cache, pages, case, gk, gv, g):
    """keys and values of the pages, as the cache's writer leaves them"""
    H, D, PS = case["kv_heads"], case["head_dim"], case["page"]
    spikes = torch.tensor([3, D // 4 + 3, D // 2 + 3, 3 * D // 4 + 3], device="cuda")
    step = max(1, 2 ** 26 // (H * PS * D))
    for i in range(0, pages.numel(), step):
        pg = pages[i:i + step]
        k, v = torch.randn(2, pg.numel(), H, PS, D, generator=g, device="cuda")
        k[..., spikes] *= OUTLIER
        k = (k / gk).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if case["k8"] else _quantise(k, gk)
        v = _quantise(v, gv)
        cache[pg] = torch.cat((k, v), dim=3 if case["k8"] else 1)


def _hadamard(D):
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    while h.shape[0] < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h * D ** -0.5


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 23)
    H, D, G, PS = case["kv_heads"], case["head_dim"], case["group"], case["page"]
    reqs = _requests(case)
    order = torch.randperm(len(reqs), generator=torch.Generator().manual_seed(seed + 5)).tolist()
    reqs = [reqs[i] for i in order]
    B, T = len(reqs), sum(q for q, _ in reqs)
    slot = D + D // 2 + D // 16 if case["k8"] else D // 2 + D // 16
    heads = H if case["k8"] else 2 * H
    # pages: those with a token that some row sees; the eviction's new pages behind them
    MP = max((L + PS - 1) // PS for _, L in reqs)
    have = torch.zeros((B, MP), dtype=torch.bool)
    for b, (q, L) in enumerate(reqs):
        lo = _first_seen(case, q, L)
        have[b, lo // PS:(L + PS - 1) // PS] = True
        have[b, :(min(lo, case["sinks"]) + PS - 1) // PS] = True
    total = int(have.sum())
    n_out = B * ((case["keep"] + PS - 1) // PS) if case["op"] == "evict" else 0
    if case["order"] == "LBNHC":
        phys = torch.zeros((1 + total + n_out, PS, heads, slot), dtype=torch.uint8, device="cuda")
        cache = phys.permute(0, 2, 1, 3)
    else:
        phys = cache = torch.zeros((1 + total + n_out, heads, PS, slot), dtype=torch.uint8, device="cuda")
    phys[0] = 0xff
    pool = torch.randperm(total, generator=g, device="cuda") + 1
    bt = torch.zeros((B, MP), dtype=torch.int32, device="cuda")
    bt[have.cuda()] = pool.to(torch.int32)
    gk = OUTLIER * 5.5 / (448 if case["k8"] else 6 * 448)
    gv = 5.5 / (6 * 448)
    _fill(cache, pool, case, gk, gv, g)
    flat_of = phys.view(-1)
    parts = (0, D, D, D + D // 2) if case["k8"] else (0, D // 2, H * cache.stride(1), H * cache.stride(1) + D // 2)
    st = (cache.stride(0), cache.stride(2), cache.stride(1))
    s = SimpleNamespace(op=case["op"], B=B, H=H, G=G, D=D, page=PS, k8=case["k8"], had=case["had"], phys=phys, cache=cache, bt=bt,
                        flat=tuple(flat_of[p:] for p in parts), strides=st + st, sm=D ** -0.5, gk_value=gk, gv_value=gv,
                        gk=torch.full((H,), gk, device="cuda"), gv=torch.full((H,), gv, device="cuda"), window=case.get("window", 0),
                        sinks=case["sinks"], lens=torch.tensor([L for _, L in reqs], dtype=torch.int32, device="cuda"), ws=None, signs=None,
                        table=torch.tensor(_E2M1, device="cuda"))
    if case["op"] == "evict":
        s.keep, s.recent = case["keep"], case["recent"]
        W = max(L for _, L in reqs)
        w = torch.exp(2 * torch.randn(B, H, W, generator=g, device="cuda"))
        s.weights = w * (torch.rand(B, H, W, generator=g, device="cuda") > 0.1)
        s.first_out = 1 + total
        new = torch.randperm(n_out, generator=g, device="cuda") + s.first_out
        s.out_bt = new.to(torch.int32).view(B, -1)
        s.kept = torch.zeros((B, H, s.keep), dtype=torch.int32, device="cuda")
        s.out_lens = torch.zeros((B,), dtype=torch.int32, device="cuda")
        s.out_weights = torch.zeros((B, H, s.keep), device="cuda")
        return s
    s.qlens = [q for q, _ in reqs]
    s.qlmax = max(s.qlens)
    s.qsl = torch.tensor([0] + s.qlens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    s.q = torch.randn(T, H * G, D, generator=g, device="cuda").to(torch.bfloat16)
    s.row_of = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(s.qlens, device="cuda"))
    s.tok_of = torch.arange(T, device="cuda") - s.qsl[s.row_of].long()
    s.q_len = torch.tensor(s.qlens, device="cuda")
    s.reach = (max(L for _, L in reqs) if not s.window else min(max(L for _, L in reqs), s.window + s.qlmax - 1))
    if case["had"]:
        s.signs = (torch.randint(0, 2, (D,), generator=torch.Generator().manual_seed(0x6B7634)) * 2 - 1).float().cuda()
        s.hadamard = _hadamard(D)
    s.rows = [(b, a, a + q, L) for b, (a, (q, L)) in enumerate(zip(s.qsl.tolist(), reqs))]
    s.lse = None
    if case["op"] == "weights":
        s.lse = torch.zeros(T, H * G, device="cuda")
        for b, a, e, L in s.rows:                     # the log-sum-exps that the attention before has left
            x, _, see = _scores64(s, b, a, e, L)
            s.lse[a:e] = torch.logsumexp(x.masked_fill(~see, -math.inf), -1).permute(1, 0, 2).reshape(e - a, H * G).float()
        s.weights = 1e-3 * torch.rand(B, H, max(L for _, L in reqs), generator=g, device="cuda")     # of a few steps before
    else:
        s.out = torch.zeros_like(s.q)
        if case["lse"]:
            s.lse = torch.zeros(T, H * G, device="cuda")
    return s


# --------------------------------------------------------------------------------------------------------- plain forms
def _values(s, b):
    """codes two to a byte with block scales behind them, (.., D / 2 + D / 16) bytes -> (.., D) fp32"""
    D = s.D
    code = torch.stack((b[..., :D // 2] & 15, b[..., :D // 2] >> 4), dim=-1)
    sf = b[..., D // 2:].contiguous().view(torch.float8_e4m3fn).float()
    x = s.table.index_select(0, code.reshape(-1).int()).view(*b.shape[:-1], D // 16, 16)
    return (x * sf[..., None]).reshape(*b.shape[:-1], D)


def _seen_keys(s, with_values):
    """positions (B, N) that some row of a request sees, which of them exist, and the keys (and values) there, (B, H, N, D) fp32"""
    dev, L = "cuda", s.lens.long()
    near = L[:, None] - s.reach + torch.arange(s.reach, device=dev)
    first = L - s.q_len - s.window + 1 if s.window else torch.zeros_like(L)
    sinks = s.sinks if s.window else 0
    ok = near >= first.clamp(min=sinks)[:, None]
    far = torch.arange(sinks, device=dev).expand(s.B, -1)
    pos = torch.cat((far, near), 1)
    ok = torch.cat((far < L[:, None], ok), 1)
    at = pos.clamp(min=0).minimum(L[:, None] - 1)
    page = torch.gather(s.bt.long(), 1, at // s.page)
    slots = s.cache[page, :, at % s.page].permute(0, 2, 1, 3)              # (B, heads, N, slot)
    if s.k8:
        k = slots[..., :s.D].contiguous().view(torch.float8_e4m3fn).float()
        v = _values(s, slots[..., s.D:]) if with_values else None
    else:
        k = _values(s, slots[:, :s.H])
        v = _values(s, slots[:, s.H:]) if with_values else None
    return pos, ok, k, v


def _plain_scores(s, pos, ok, k):
    """scores (B, H, qlmax * G, N) with -inf where a row does not see a key, and where the rows of the batch lie in it"""
    q = s.q.float()
    if s.had:
        q = ((s.q.double() * s.signs) @ s.hadamard).to(torch.bfloat16).float()
    qp = torch.zeros(s.B, s.H, s.qlmax, s.G, s.D, device="cuda")
    qp[s.row_of, :, s.tok_of] = q.view(-1, s.H, s.G, s.D)
    x = qp.view(s.B, s.H, s.qlmax * s.G, s.D) @ (k * (s.sm * s.gk_value)).transpose(2, 3)
    p = (s.lens.long() - s.q_len)[:, None] + torch.arange(s.qlmax, device="cuda")          # positions of the query tokens
    see = ok[:, None, :] & (pos[:, None, :] <= p[:, :, None])
    if s.window:
        see &= (pos[:, None, :] > p[:, :, None] - s.window) | (pos[:, None, :] < s.sinks)
    see &= (torch.arange(s.qlmax, device="cuda") < s.q_len[:, None])[:, :, None]
    see = see[:, None, :, None, :].expand(-1, s.H, -1, s.G, -1).reshape(x.shape)
    return torch.where(see, x, -math.inf)


def _plain_attention(s):
    pos, ok, k, v = _seen_keys(s, True)
    x = _plain_scores(s, pos, ok, k)
    del k
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = (x - m).exp()
    den = e.sum(-1, keepdim=True)
    o = e @ torch.where(ok[:, None, :, None], v, 0.0) / torch.where(den > 0, den, 1.0) * s.gv_value
    shape = (s.B, s.H, s.qlmax, s.G)
    s.out.copy_(o.view(*shape, s.D)[s.row_of, :, s.tok_of].reshape(s.out.shape))
    if s.lse is not None:
        s.lse.copy_((m + den.log()).view(shape)[s.row_of, :, s.tok_of].reshape(s.lse.shape))


def _plain_weights(s):
    pos, ok, k, _ = _seen_keys(s, False)
    x = _plain_scores(s, pos, ok, k)
    lse = torch.zeros(s.B, s.H, s.qlmax, s.G, device="cuda")
    lse[s.row_of, :, s.tok_of] = s.lse.view(-1, s.H, s.G)
    w = (x - lse.view(s.B, s.H, -1, 1)).exp().sum(2)
    at = torch.where(ok, pos, 0)[:, None, :].expand(-1, s.H, -1)
    s.weights.scatter_add_(2, at, torch.where(ok[:, None], w, 0.0))


def _plain_evict(s):
    L = s.lens.long()
    W = s.weights.shape[2]
    col = torch.arange(max(W, s.keep), device="cuda")
    w = torch.nn.functional.pad(s.weights, (0, max(0, s.keep - W)))
    there = col < L[:, None]
    stay = (col < s.sinks) | (col >= L[:, None] - s.recent)
    w = torch.where(stay[:, None], math.inf, w)
    w = torch.where(there[:, None], w, -math.inf)
    n = L.clamp(max=s.keep)
    first = w.sort(dim=2, descending=True, stable=True).indices[..., :s.keep].sort(dim=2).values
    on = (torch.arange(s.keep, device="cuda") < n[:, None])[:, None].expand_as(first)
    s.kept.copy_(torch.where(on, first, -1))
    s.out_lens.copy_(n)
    at = first.minimum(L[:, None, None] - 1)
    s.out_weights.copy_(torch.where(on, s.weights.gather(2, at), s.out_weights))
    b = torch.arange(s.B, device="cuda")[:, None, None]
    r = torch.arange(s.keep, device="cuda")
    page, new = s.bt.long()[b, at // s.page], torch.where(on, s.out_bt.long()[:, None, r // s.page], 0)      # (page 0: a dump)
    h = torch.arange(s.H, device="cuda")[None, :, None]
    s.cache[new, h, (r % s.page).expand_as(at)] = s.cache[page, h, at % s.page]
    if not s.k8:
        s.cache[new, s.H + h, (r % s.page).expand_as(at)] = s.cache[page, s.H + h, at % s.page]


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


def run(state):
    s = state
    if s.op == "decode":
        if own:
            _kernels().decode_window(s.q, s.flat, s.strides, s.page, s.bt, s.lens, s.qsl, s.sm, 1.0, s.gk, s.gv, s.qlmax, s.out,
                                     _workspace(s), s.window, s.sinks, signs=s.signs, k8=s.k8, lse=s.lse)
        else:
            _plain_attention(s)
        return {"out": s.out, "lse": s.lse}
    if s.op == "prefill":
        if own:
            _kernels().prefill_window(s.q, s.flat, s.strides, s.page, s.bt, s.rows, s.sm * s.gk_value, s.gv_value, s.H, s.out, s.window,
                                      s.sinks, signs=s.signs, k8=s.k8, workspace=_workspace(s), lse=s.lse)
        else:
            _plain_attention(s)
        return {"out": s.out, "lse": s.lse}
    if s.op == "weights":
        if own:
            _kernels().accumulate_weights(s.q, s.flat, s.strides, s.page, s.bt, s.lens, s.qsl, s.sm, s.gk, s.qlmax, s.lse, s.weights,
                                          window=s.window, sinks=s.sinks, signs=s.signs, k8=s.k8)
        else:
            _plain_weights(s)
        return {"weights": s.weights}
    if own:
        _kernels().evict(s.flat, s.strides, s.page, s.D, s.bt, s.lens, s.weights, s.keep, s.sinks, s.recent, s.kept, s.out_lens,
                         out_tables=s.out_bt, out_weights=s.out_weights, k8=s.k8)
    else:
        _plain_evict(s)
    return {"kept": s.kept, "lens": s.out_lens, "weights": s.out_weights, "cache": s.phys[s.first_out:]}


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    H, D, PS = case["kv_heads"], case["head_dim"], case["page"]
    HQ = H * case["group"]
    slot = D + D // 2 + D // 16 if case["k8"] else 2 * (D // 2 + D // 16)       # cached bytes of a token and kv head
    key = D if case["k8"] else D // 2 + D // 16
    n = flops = 0
    for q, L in _requests(case):
        if case["op"] == "evict":
            keep = min(L, case["keep"])
            n += H * (4 * L + keep * (2 * slot + 8)) + 4 * ((L + PS - 1) // PS + (keep + PS - 1) // PS) + 8
            continue
        seen = _seen(case, q, L)
        pairs = sum(_pairs(case, L - q + t) for t in range(q))
        rows = q * HQ
        n += 4 * (seen + PS - 1) // PS + 12
        if case["op"] == "weights":
            n += seen * H * (key + 8) + rows * (2 * D + 4)
            flops += 2 * D * HQ * pairs
        else:
            n += seen * H * slot + rows * (4 * D + 4 * case["lse"])
            flops += 4 * D * HQ * pairs
    return {"bytes": n, "flops": flops}


def _pairs(case, p):
    """keys that the query token at position p sees"""
    lo = max(0, p - case["window"] + 1) if case["window"] else 0
    return p + 1 - lo + min(lo, case["sinks"])


# --------------------------------------------------------------------------------------------------------------- exact
def _slots64(s, b, h, side, pos):
    """side 0: keys, 1: values of head h at the positions, in 64 bits"""
    page = s.bt[b, pos // s.page].long()
    raw = s.cache[page, h if s.k8 or side == 0 else s.H + h, pos % s.page]
    if s.k8:
        if side == 0:
            return raw[:, :s.D].contiguous().view(torch.float8_e4m3fn).double()
        raw = raw[:, s.D:]
    code = torch.empty((raw.shape[0], s.D), dtype=torch.int64, device="cuda")
    code[:, 0::2] = raw[:, :s.D // 2] % 16
    code[:, 1::2] = raw[:, :s.D // 2] // 16
    mag, sign = code % 8, 1 - 2 * (code // 8)
    # E2M1: one mantissa bit, exponent bias 1, subnormal steps of a half
    val = torch.where(mag < 2, mag * 0.5, (1 + (mag % 2) * 0.5) * 2.0 ** (mag // 2 - 1).double())
    sf = raw[:, s.D // 2:].contiguous().view(torch.float8_e4m3fn).double()
    return sign * val * sf.repeat_interleave(16, dim=1)


def _scores64(s, b, a, e, L):
    """scores (H, e - a, G, N) of request b's rows a .. e - 1 against the positions (N) that some of them sees, in 64 bits, and
    who sees what"""
    lo = max(0, L - (e - a) - s.window + 1) if s.window else 0
    pos = torch.cat((torch.arange(min(lo, s.sinks), device="cuda"), torch.arange(lo, L, device="cuda")))
    q = s.q[a:e].double().view(e - a, s.H, s.G, s.D)
    if s.had:
        q = ((q * s.signs.double()) @ s.hadamard).to(torch.bfloat16).double()
    x = torch.stack([q[:, h] @ _slots64(s, b, h, 0, pos).T for h in range(s.H)]) * (s.sm * s.gk_value)
    p = torch.arange(L - (e - a), L, device="cuda")[:, None]
    see = pos[None] <= p
    if s.window:
        see &= (p - pos[None] < s.window) | (pos[None] < s.sinks)
    return x, pos, see[None, :, None, :]


def exact(case, seed):
    """Every operator from its definition in 64 bits: attention and log-sum-exp row by row, the weights summed over the rows,
    the weights that an eviction keeps. The eviction's whole numbers and bytes have no value here."""
    s = prepare(case, seed)
    H, G = s.H, s.G
    if s.op == "evict":
        w = s.weights.double().cpu()
        new = torch.zeros(s.B, H, s.keep, dtype=torch.float64)
        for b, L in enumerate(s.lens.tolist()):
            for h in range(H):
                x = w[b, h, :L]
                if L > s.keep:
                    mid = torch.arange(s.sinks, L - s.recent)
                    best = mid[torch.sort(-x[mid], stable=True).indices[:s.keep - s.sinks - s.recent]]
                    stay = torch.zeros(L, dtype=torch.bool)
                    stay[:s.sinks] = True
                    stay[L - s.recent:] = True
                    stay[best] = True
                    x = x[stay]
                new[b, h, :x.numel()] = x
        return {"kept": None, "lens": None, "weights": new.cuda(), "cache": None}
    if s.op == "weights":
        new = s.weights.double()
        for b, a, e, L in s.rows:
            x, pos, see = _scores64(s, b, a, e, L)
            x = x - s.lse[a:e].double().view(e - a, H, G).permute(1, 0, 2)[..., None]
            new[b][:, pos] += torch.where(see, x.exp(), 0.0).sum((1, 2))
        return {"weights": new}
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s.q.shape[:2], dtype=torch.float64, device="cuda")
    for b, a, e, L in s.rows:
        step = max(1, 2 ** 29 // (H * G * L))                    # (query tokens at a time)
        for t in range(a, e, step):
            u = min(e, t + step)
            n = L - (e - u)                                      # the context as the last of these tokens sees it
            x, pos, see = _scores64(s, b, t, u, n)
            x = x.masked_fill(~see, -math.inf)
            l = torch.logsumexp(x, -1)
            p = (x - l[..., None]).exp()
            for h in range(H):
                out[t:u, h * G:(h + 1) * G] = p[h] @ _slots64(s, b, h, 1, pos) * s.gv_value
            lse[t:u] = l.permute(1, 0, 2).reshape(u - t, H * G)
    return {"out": out, "lse": lse if s.lse is not None else None}
