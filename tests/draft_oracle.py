"""Plain 64-bit restatements of the operators around a decode step with drafted tokens, and how far a result in fewer bits may be from them."""
import math

import torch


def depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def sees(parents):
    """[S, S]: row i sees column j when j is i or one of its ancestors."""
    s = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i in range(len(parents)):
        j = i
        while j >= 0:
            s[i, j] = True
            j = parents[j]
    return s


def tree_attention(q, keys, values, table, pasts, trees, size, scale, cap, half_step):
    """Rows of trees: packed rotated queries q [T, N, H] (64 bits) over caches [blocks, size, Nk, H], which hold the new entries too.
    Returns the result and, per element, a bound on what rounding may change.

    With u the half step of the type: a rounded query moves a score by at most e_j = scale u sum_d |q_d k_d| (a cap's slope is at most 1); a weight
    rounded to the type changes by a factor within 1 +- u; 32-bit sums, exponentials and maxima add 2^-18 for scores below 2^5, as those of the
    cases are.  A weight p_j so carries a factor e^(+-n_j) with n_j = e_j + u + 2^-18, the normalised result moves by at most
    sum_j p_j (|v_j| + |o|) (e^n - 1) with n the largest of the n_j, and its own rounding adds u |o|."""
    T, N, H = q.shape
    group = N // keys.shape[2]
    out, bound, t0 = torch.zeros(T, N, H, dtype=torch.float64), torch.zeros(T, N, H, dtype=torch.float64), 0
    for b, (past, parents) in enumerate(zip(pasts, trees)):
        new = len(parents)
        if new == 0:
            continue
        where = torch.arange(past + new)
        block = table[b].long()[where // size]
        hidden = torch.cat([torch.zeros(new, past, dtype=torch.bool), ~sees(parents)], 1)
        for h in range(N):
            k, v = keys[block, where % size, h // group].double(), values[block, where % size, h // group].double()
            qh = q[t0:t0 + new, h]
            s = qh @ k.T * scale
            e = scale * half_step * (qh.abs() @ k.abs().T)
            if cap:
                s = cap * torch.tanh(s / cap)
            p = s.masked_fill(hidden, -math.inf).softmax(-1)
            o = p @ v
            n = (e.masked_fill(hidden, 0).amax(-1, keepdim=True) + half_step + 2.0 ** -18).expm1()
            out[t0:t0 + new, h] = o
            bound[t0:t0 + new, h] = n * (p @ v.abs() + o.abs()) * 1.01 + half_step * o.abs() + 1e-7
        t0 += new
    return out, bound


def process_logits(x, text, counted, repetition=1.0, presence=0.0, frequency=0.0, biases=(), allowed=None, temperature=1.0):
    """One row, 64 bits.  text: its tokens; counted: those that count for presence and frequency; biases: (token, value) pairs; allowed: tokens or
    None.  Returns the scores and a bound: every 32-bit operation rounds by u = 2^-24 of what it returns - the product or quotient of the
    repetition, frequency times count, its sum with the presence, the difference, each sum of biases and their addition, the quotient of the temperature
    - and a division by the temperature scales what came before."""
    u, V = 2.0 ** -24, len(x)
    x, off = x.double().clone(), torch.zeros(V, dtype=torch.float64)
    inside = lambda tokens: [t for t in tokens if 0 <= t < V]  # noqa: E731
    for t in set(inside(text)):
        x[t] = x[t] * repetition if x[t] < 0 else x[t] / repetition
        off[t] += u * x[t].abs()
    count = {}
    for t in inside(counted):
        count[t] = count.get(t, 0) + 1
    for t, c in count.items():
        x[t] -= frequency * c + presence
        off[t] += u * (2 * (abs(frequency * c) + abs(presence)) + x[t].abs())
    sums = {}
    for t, v in biases:
        if 0 <= t < V:
            sums.setdefault(t, []).append(v)
    for t, values in sums.items():
        x[t] += math.fsum(values) if all(map(math.isfinite, values)) else sum(values)
        off[t] += u * (len(values) * sum(map(abs, values)) + x[t].abs())
    if allowed is not None:
        keep = torch.zeros(V, dtype=torch.bool)
        keep[inside(allowed)] = True
        x[~keep] = -math.inf
    if temperature > 0 and temperature != 1:
        x, off = x / temperature, off / temperature + u * (x / temperature).abs()
    return x, torch.where(x.isfinite(), off * 1.01 + 1e-38, 0.0)
