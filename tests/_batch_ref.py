"""64-bit restatements of the batched-decode operators (rotary append,
attention behind a shared prefix, eviction) for the tests."""
import math

import torch

F64 = torch.float64


def freqs(rot, theta=1e4, scaling="none", factor=1.0, orig_ctx=0.0, turns_fast=32.0, turns_slow=1.0):
    f = torch.tensor([theta ** (-2.0 * d / rot) for d in range(rot // 2)], dtype=F64)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        g = ((orig_ctx * f / (2 * math.pi) - turns_slow) / (turns_fast - turns_slow)).clamp(0.0, 1.0)
        f = f * (g + (1.0 - g) / factor)
    return f


def rotate(x, pos, f, layout, mscale=1.0):
    """x [T][heads][hd] float64 -> (rotated, the error scale |x0| + |x1| of each element)."""
    rot = 2 * len(f)
    ang = pos.to(F64)[:, None, None] * f
    c, s = torch.cos(ang) * mscale, torch.sin(ang) * mscale
    i0, i1 = ((slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half"
              else (slice(0, rot, 2), slice(1, rot, 2)))
    y, mag = x.clone(), torch.zeros_like(x)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    mag[..., i0] = mag[..., i1] = (a.abs() + b.abs()) * mscale
    return y, mag


def attention(q, k, v, lens, n_head, n_kv, pk=None, pv=None, scale=None):
    """q [B][n_head*hd], k, v [B][C][n_kv*hd], pk, pv [L][n_kv*hd] on the CPU.
    Returns out [B][n_head*hd], the own rows' weights summed per KV head
    [B][n_kv][C], and for the error bounds sum_j p_j |v_j| like out, and per
    (b, head) the largest scale * sum_d |q_d k_d|."""
    B, C = k.shape[:2]
    hd, g = q.shape[1] // n_head, n_head // n_kv
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(B, n_head, hd, dtype=F64)
    mag, top = torch.zeros_like(out), torch.zeros(B, n_head, dtype=F64)
    w = torch.zeros(B, n_kv, C, dtype=F64)
    L = 0 if pk is None else pk.shape[0]
    for b in range(B):
        n = int(lens[b])
        if L + n == 0:
            continue
        for h in range(n_head):
            c = slice(h // g * hd, (h // g + 1) * hd)
            kk, vv = k[b, :n, c].to(F64), v[b, :n, c].to(F64)
            if L:
                kk, vv = torch.cat([pk[:, c].to(F64), kk]), torch.cat([pv[:, c].to(F64), vv])
            qq = q[b, h * hd:(h + 1) * hd].to(F64)
            p = torch.softmax(scale * (kk @ qq), 0)
            out[b, h], mag[b, h] = p @ vv, p @ vv.abs()
            top[b, h] = abs(scale) * (kk.abs() @ qq.abs()).max()
            w[b, h // g, :n] += p[L:]
    return out.view(B, -1), w, mag.view(B, -1), top


def evict(lens, pos, w, keep, n_sink, n_recent):
    """Per (b, g) the (place, mover) pairs, with new lens, pos and w."""
    lens, pos, w = lens.clone(), pos.clone(), w.clone()
    moves = {}
    B, G, C = pos.shape
    for b in range(B):
        n = int(lens[b])
        if n <= keep or n > C:
            continue
        for g in range(G):
            p, x = pos[b, g, :n].tolist(), w[b, g, :n].tolist()
            newest = max(p)

            def rank(i):
                safe = p[i] < n_sink or p[i] > newest - n_recent
                bad = x[i] != x[i]
                return (not safe, bad and not safe, 0.0 if safe or bad else -x[i], i)

            kept = set(sorted(range(n), key=rank)[:keep])
            pairs = list(zip([i for i in range(keep) if i not in kept], [i for i in range(keep, n) if i in kept]))
            for d, s in pairs:
                pos[b, g, d], w[b, g, d] = pos[b, g, s], w[b, g, s]
            w[b, g, keep:n] = 0.0
            moves[b, g] = pairs
        lens[b] = keep
    return lens, pos, w, moves


def apply_moves(t, moves, n_kv):
    """t [B][C][n_kv*hd]: the rows of the pairs moved."""
    t = t.clone()
    v = t.view(t.shape[0], t.shape[1], n_kv, -1)
    for (b, g), pairs in moves.items():
        for d, s in pairs:
            v[b, d, g] = v[b, s, g]
    return t
