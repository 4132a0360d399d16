"""Plain 64-bit forms of the multi-axis rotation, the block means, the block
lists and the attention over them, on torch CPU tensors (float64 or int64)."""
import math

import torch


def angles(pos, dims, scales, theta, one_progression, head_dim):
    """[seq, head_dim / 2] angles in radians."""
    out = torch.zeros(pos.shape[0], head_dim // 2, dtype=torch.float64)
    j = 0
    for a, dim in enumerate(dims):
        for i in range(dim // 2):
            power = 2.0 * j / head_dim if one_progression else 2.0 * i / dim
            out[:, j] = pos[:, a].double() * ((scales[a] if scales else 1.0) * theta ** -power)
            j += 1
    return out


def norm_rope(x, heads, head_dim, w, eps, ang, split_half):
    """Result and, per element, the sum of the magnitudes its rotation adds."""
    x = x.double().reshape(x.shape[0], heads, head_dim)
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    c, s = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    half = head_dim // 2
    i0 = torch.arange(half) if split_half else 2 * torch.arange(half)
    i1 = i0 + half if split_half else i0 + 1
    y, mag = torch.empty_like(x), torch.empty_like(x)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    mag[..., i0] = mag[..., i1] = a.abs() + b.abs()
    return y.reshape(x.shape[0], -1), mag.reshape(x.shape[0], -1)


def means(x, heads, head_dim, block, mask=None):
    """(means [n, heads, head_dim], counts [n], mean magnitudes [n, heads, head_dim])."""
    seq = x.shape[0]
    n = (seq + block - 1) // block
    m, mag = torch.zeros(n, heads * head_dim, dtype=torch.float64), torch.zeros(n, heads * head_dim, dtype=torch.float64)
    counts = torch.zeros(n, dtype=torch.int32)
    for b in range(n):
        rows = torch.arange(b * block, min(seq, (b + 1) * block))
        if mask is not None:
            rows = rows[mask[rows] != 0]
        counts[b] = rows.numel()
        if rows.numel():
            m[b], mag[b] = x[rows].double().mean(0), x[rows].double().abs().mean(0)
    shape = (n, heads, head_dim)
    return m.reshape(shape), counts, mag.reshape(shape)


def select(qm, km, counts, topk, keep_first, keep_last):
    """[heads, q_blocks, topk] int32, by the definition, one row at a time."""
    nq, heads = qm.shape[:2]
    nk, kv = km.shape[:2]
    out = torch.full((heads, nq, topk), -1, dtype=torch.int32)
    for h in range(heads):
        score = qm[:, h].double() @ km[:, h // (heads // kv)].double().T if nk else torch.zeros(nq, 0)
        for i in range(nq):
            row = [-math.inf if math.isnan(v) else v for v in score[i].tolist()]
            usable = [j for j in range(nk) if counts is None or counts[j] > 0]
            always = [j for j in usable if j < keep_first or j >= nk - keep_last]
            rest = sorted((j for j in usable if j not in always), key=lambda j: (-row[j], j))
            found = sorted(always + rest[:topk - len(always)])
            out[h, i, :len(found)] = torch.tensor(found, dtype=torch.int32)
    return out


def attention(q, k, v, heads, kv_heads, head_dim, scale, mask, lists, q_block, k_block):
    """(out, sum of p |v|), both [seq_q, heads * head_dim]."""
    seq_q, seq_k = q.shape[0], k.shape[0]
    nk = (seq_k + k_block - 1) // k_block
    out = torch.zeros(seq_q, heads * head_dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for h in range(heads):
        g = h // (heads // kv_heads)
        cols, kcols = slice(h * head_dim, (h + 1) * head_dim), slice(g * head_dim, (g + 1) * head_dim)
        for i in range((seq_q + q_block - 1) // q_block):
            keys = [r for b in lists[h, i].tolist() if 0 <= b < nk
                    for r in range(b * k_block, min(seq_k, (b + 1) * k_block)) if mask is None or mask[r] != 0]
            if not keys:
                continue
            rows = slice(i * q_block, min(seq_q, (i + 1) * q_block))
            kk, vv = k[keys][:, kcols].double(), v[keys][:, kcols].double()
            p = torch.softmax(scale * (q[rows, cols].double() @ kk.T), dim=1)
            out[rows, cols] = p @ vv
            mag[rows, cols] = p @ vv.abs()
    return out, mag
