"""Plain 64-bit restatements of the serving operators, and how far a result in fewer bits may be from them."""
import math

import torch


def blocks_of(tokens, size):
    return -(-tokens // size)


def batch_layout(past, new, table, free, rows, size):
    """(table, cumulative lengths, positions, slots, blocks used) as lists; a batch that does not fit leaves the table as it is."""
    table = [list(r) for r in table]
    cum, pos, slot = [0] * (len(past) + 1), [-1] * rows, [-1] * rows
    pairs = list(zip(past, new))
    need = sum(blocks_of(p + n, size) - blocks_of(p, size) for p, n in pairs)
    if any(p < 0 or n < 0 for p, n in pairs):
        return table, cum, pos, slot, -4
    if sum(new) > rows:
        return table, cum, pos, slot, -3
    if any(n > 0 and blocks_of(p + n, size) > len(table[0]) for p, n in pairs):
        return table, cum, pos, slot, -2
    if need > len(free):
        return table, cum, pos, slot, -1
    free, t = list(free), 0
    for b, (p, n) in enumerate(pairs):
        for j in range(blocks_of(p, size), blocks_of(p + n, size)):
            table[b][j] = free.pop(0)
        for s in range(n):
            pos[t], slot[t] = p + s, table[b][(p + s) // size] * size + (p + s) % size
            t += 1
        cum[b + 1] = t
    return table, cum, pos, slot, need


def rotate(x, cos, sin, interleaved=False):
    """x [rows, heads, H], cos and sin [rows, r / 2]: the first r elements of every head turn."""
    half = cos.shape[1]
    y, cos, sin = x.clone(), cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    u, v = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = u, v
    else:
        y[..., :half], y[..., half:2 * half] = u, v
    return y


def paged_attention(q, keys, values, table, lengths, size, scale, cap, half_step):
    """Causal attention of packed rotated queries q [T, N, H] (64 bits) over caches [blocks, size, Nk, H]; lengths: (past, new) per
    sequence.  Returns the result and, per element, a bound on what rounding may change:

    with u the half step of the type, a rounded query moves a score by at most e_j = scale u sum_d |q_d k_d| (a cap's slope is at
    most 1), a weight rounded to the type changes by a factor within 1 +- u, and 32-bit sums, exponentials and maxima add 2^-18
    in all for scores below 2^5.  So every weight p_j carries a factor e^(+-n_j), n_j = e_j + u + 2^-18, the normalised result moves by at most
    sum_j p_j (|v_j| + |o|) (e^(n) - 1) with n = max n_j, and its own rounding adds u |o|.  (Scores of the cases stay below 2^5.)"""
    T, N, H = q.shape
    Nk = keys.shape[2]
    out, bound, t0 = torch.zeros(T, N, H, dtype=torch.float64), torch.zeros(T, N, H, dtype=torch.float64), 0
    for b, (past, new) in enumerate(lengths):
        if new == 0:
            continue
        where = torch.arange(past + new)
        block = table[b].long()[where // size]
        for h in range(N):
            k, v = keys[block, where % size, h // (N // Nk)].double(), values[block, where % size, h // (N // Nk)].double()
            qh = q[t0:t0 + new, h]
            s = qh @ k.T * scale
            e = scale * half_step * (qh.abs() @ k.abs().T)
            if cap:
                s = cap * torch.tanh(s / cap)
            hidden = where > torch.arange(past, past + new).unsqueeze(1)
            p = s.masked_fill(hidden, -math.inf).softmax(-1)
            o = p @ v
            n = (e.masked_fill(hidden, 0).amax(-1, keepdim=True) + half_step + 2.0 ** -18).expm1()
            out[t0:t0 + new, h] = o
            bound[t0:t0 + new, h] = n * (p @ v.abs() + o.abs()) * 1.01 + half_step * o.abs() + 1e-7
        t0 += new
    return out, bound


def token_log_probs(x, tokens, k):
    """(log probability, entropy, log probabilities and indices of the k largest, log sum exp) of 64-bit logits [rows, vocab]."""
    rows, V = x.shape
    out = [torch.zeros(rows, dtype=torch.float64) for _ in range(3)]
    top, index = torch.zeros(rows, k, dtype=torch.float64), torch.zeros(rows, k, dtype=torch.int64)
    for r in range(rows):
        row = [float(v) for v in x[r]]
        order = sorted(range(V), key=lambda v: (-math.inf if math.isnan(row[v]) else -row[v], v))[:k] if not any(map(math.isnan, row)) else \
            sorted(range(V), key=lambda v: (0 if math.isnan(row[v]) else 1, -row[v] if not math.isnan(row[v]) else 0.0, v))[:k]
        index[r] = torch.tensor(order, dtype=torch.int64)
        bad = any(math.isnan(v) or v == math.inf for v in row)
        m = max(row)
        if bad or m == -math.inf:
            lse, entropy = (math.nan, math.nan) if bad else (-math.inf, 0.0)
        else:
            s = math.fsum(math.exp(v - m) for v in row)
            lse = m + math.log(s)
            entropy = -math.fsum(math.exp(v - lse) * (v - lse) for v in row if v != -math.inf)
        of = lambda v: math.nan if bad else (-math.inf if m == -math.inf else row[v] - lse)  # noqa: E731
        tok = int(tokens[r])
        out[0][r] = of(tok) if 0 <= tok < V else 0.0
        out[1][r], out[2][r] = entropy, lse
        top[r] = torch.tensor([of(v) for v in order], dtype=torch.float64)
    return out[0], out[1], top, index, out[2]


def token_log_probs_grad(x, tokens, g_lp, g_h, index, g_top, g_lse):
    """Gradient of sum g_lp log_prob + g_h entropy + g_top top_log_probs + g_lse log_sum_exp, [rows, vocab], from the definitions."""
    rows, V = x.shape
    dx = torch.zeros_like(x)
    for r in range(rows):
        if (x[r] == -math.inf).all():
            continue
        p = x[r].softmax(-1)
        logp = torch.log_softmax(x[r], -1)
        entropy = -torch.special.xlogy(p, p).sum()
        unit = lambda v: torch.nn.functional.one_hot(torch.tensor(int(v)), V).double()  # noqa: E731
        if 0 <= int(tokens[r]) < V:
            dx[r] += g_lp[r] * (unit(tokens[r]) - p)
        dx[r] -= g_h[r] * torch.where(p > 0, p * (torch.where(p > 0, logp, 0.0) + entropy), 0.0)
        for j in range(index.shape[1]):
            dx[r] += g_top[r, j] * (unit(index[r, j]) - p)
        dx[r] += g_lse[r] * p
    return dx
