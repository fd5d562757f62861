"""Plain 64-bit forms of the operators for bounded caches, on the CPU: attention over a sliding window and the first tokens,
the weights that keys gather, and the eviction that goes by them. Written from the definitions, without the kernels' layout."""
import numpy as np
import torch

from horizon_kernels_b200 import layout as Lt

E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def e4m3(b):
    return b.contiguous().view(torch.float8_e4m3fn).double()


def fp4(data, sf):
    """(.., D / 2) code bytes and (.., D / 16) scale bytes -> (.., D)"""
    code = torch.stack((data & 15, data >> 4), dim=-1).reshape(*data.shape[:-1], -1).long()
    return E2M1[code] * e4m3(sf).repeat_interleave(16, dim=-1)


def views(phys, kind, KVH, D):
    """[page, position, head, byte] views of a cache tensor in one of the layouts"""
    if kind == "region":
        return Lt.split_views(phys, KVH)
    if kind == "k8":
        return Lt.k8_views(phys, D)
    return Lt.slot_views(phys.permute(0, 2, 1, 3) if kind == "nhd" else phys, KVH, D)


def token(view, row, PS, j):
    """(positions j of a request, heads, bytes) of one part"""
    return view[row[j // PS].long(), j % PS]


def dense(phys, kind, KVH, D, row, PS, L, pos=None):
    """keys and values (n, KVH, D) of a request's positions (all of them), in 64 bits, without the global scales"""
    v = [x.cpu() for x in views(phys.cpu(), kind, KVH, D)]
    j = torch.arange(L) if pos is None else pos
    row = row.cpu()
    if kind == "k8":
        return e4m3(token(v[0], row, PS, j)), fp4(token(v[1], row, PS, j), token(v[2], row, PS, j))
    return fp4(token(v[0], row, PS, j), token(v[1], row, PS, j)), fp4(token(v[2], row, PS, j), token(v[3], row, PS, j))


def seen(L, ql, window, sinks):
    """(ql, L): which keys the last ql tokens of a context of L see"""
    p = torch.arange(L - ql, L)[:, None]
    j = torch.arange(L)[None]
    see = j <= p
    if window:
        see &= (p - j < window) | (j < sinks)
    return see


def scores(q, k, scale):
    """q (ql, KVH, G, D), k (n, KVH, D) -> (ql, KVH, G, n)"""
    return torch.einsum("thgd,jhd->thgj", q.double(), k) * torch.as_tensor(scale, dtype=torch.float64).view(1, -1, 1, 1)


def attention(q, k, v, scale, vscale, window, sinks):
    """q (ql, KVH, G, D) over the first L tokens; out (ql, KVH, G, D) and the natural log-sum-exps (ql, KVH, G). scale: softmax
    scale with the keys' global ones, per head; vscale: of the output, per head"""
    L, ql = k.shape[0], q.shape[0]
    see = seen(L, ql, window, sinks)[:, None, None, :]
    x = scores(q, k, scale).masked_fill(~see, -torch.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.where(see, (x - torch.where(lse == -torch.inf, 0.0, lse)[..., None]).exp(), 0.0)
    keep = see.any(0).view(-1)                           # (a key that nobody sees may hold anything)
    out = torch.einsum("thgj,jhd->thgd", p[..., keep], v[keep]) * torch.as_tensor(vscale, dtype=torch.float64).view(1, -1, 1, 1)
    return out, lse


def gathered(q, k, scale, lse, window, sinks):
    """(KVH, L): what a call adds to the weights"""
    L, ql = k.shape[0], q.shape[0]
    see = seen(L, ql, window, sinks)[:, None, None, :]
    x = scores(q, k, scale)
    return torch.where(see, (x - lse.double()[..., None]).exp(), 0.0).sum((0, 2))


def kept_positions(w, keep, sinks, recent):
    """which of the L = len(w) tokens stay, by a plain sort"""
    L = len(w)
    if L <= keep:
        return np.arange(L)
    mid = np.arange(sinks, L - recent)
    x = np.asarray(w, np.float64)[mid]
    order = sorted(range(len(mid)), key=lambda i: (0 if np.isnan(x[i]) else 1, 0.0 if np.isnan(x[i]) else -x[i], i))
    return np.sort(np.concatenate([np.arange(sinks), mid[order[:keep - sinks - recent]], np.arange(L - recent, L)])).astype(np.int64)
