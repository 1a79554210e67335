"""Plain forms of the operators around a serving step, in 64 bits or whole numbers, for the tests."""
import math

import torch

NO_SLOT = NO_PAGE = 0xFFFFFFFF


def ids(values, shape=None):
    """Device ids: 32-bit words, given as numbers from 0 to 2^32 - 1."""
    t = torch.tensor(values, dtype=torch.int64).reshape(shape) if shape else torch.tensor(values, dtype=torch.int64)
    return torch.where(t > 2**31 - 1, t - 2**32, t).to(torch.int32).cuda()


def words(t):
    """What device ids hold, as numbers from 0 to 2^32 - 1."""
    return (t.cpu().to(torch.int64) & 0xFFFFFFFF).tolist()


def softmax_rows(q, k, v, seen, scale, k_size=None, v_size=None):
    """For q [rows, heads, d], k and v [keys, kv_heads, d] and seen [rows, keys], in 64 bits: the outputs, the weighted
    sums of |v| and the largest sum |q k| of the seen keys (or with these sizes in place of |k| and |v|). Rows that see
    nothing give zeros."""
    q, k, v = (x.double() for x in (q, k, v))
    k_size, v_size = k.abs() if k_size is None else k_size, v.abs() if v_size is None else v_size
    g = q.shape[1] // k.shape[1]
    out, mean, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for h in range(q.shape[1]):
        kk, vv = k[:, h // g], v[:, h // g]
        s = (q[:, h] @ kk.T.contiguous()) * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(dim=1, keepdim=True)
        e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        w = e / e.sum(dim=1, keepdim=True).clamp_min(1e-300)
        out[:, h], mean[:, h] = w @ vv, w @ v_size[:, h // g]
        size[:, h] = torch.where(seen, q[:, h].abs() @ k_size[:, h // g].T.contiguous(), torch.zeros_like(s)).amax(dim=1)
    return out, mean, size


def prompt_bound(out, mean, size, scale, d, n, bf16):
    """How far an output may be off: a score by d roundings of 2^-24 of sum |q k| (and a few of its product with the
    scale and in the exponential), which moves a weight by as much relative to itself; a sum over n keys by n roundings;
    with BF16 the weights by 2^-8 of each and the result by 2^-8 of itself."""
    score = (d + 16) * 2.0**-24 * abs(scale) * size[..., None] + 2.0**-21
    weight = 2 * score + (n + 16) * 2.0**-24 + (2.0**-8 if bf16 else 0.0)
    return mean * weight * 1.01 + (out.abs() * 2.0**-8 if bf16 else out.abs() * 2.0**-23) + 1e-30


def causal(n, window, device="cuda"):
    i = torch.arange(n, device=device)
    seen = i[None] <= i[:, None]
    return seen & (i[None] > i[:, None] - window) if window else seen


def plan(past, new, held, tables, free, page, prefix, width, row_tokens=0, max_tokens=None, parents=None):
    """turbo_batch_plan in plain Python: lists in, a dict of lists out (tables are changed)."""
    b = len(past)
    free, kept, missing, taken = list(free), [], 0, 0
    held = list(held)
    add = [min(n, row_tokens) if row_tokens else n for n in new]
    for i in range(b):
        need = -(-max(0, past[i] + add[i] - prefix) // page)
        got = 0
        for j in range(held[i], need):
            if j >= width:
                missing += 1
                continue
            if free:
                tables[i][j] = free.pop()
                taken += 1
                got += 1
            else:
                tables[i][j] = NO_PAGE
                missing += 1
        kept.append(held[i] + got)
    starts = [i * row_tokens for i in range(b + 1)] if row_tokens else [sum(add[:i]) for i in range(b + 1)]
    n = b * row_tokens if row_tokens else max_tokens
    positions, slots = [0] * n, [NO_SLOT] * n
    masks = [[0] * row_tokens for _ in range(b)] if parents is not None else None
    for i in range(b):
        for t in range(add[i]):
            at, pos = starts[i] + t, past[i] + t
            if at >= n:
                continue
            depth = t
            if parents is not None:
                p = parents[i][t]
                ok = p == -1 or (0 <= p < t and masks[i][p])
                masks[i][t] = ((masks[i][p] if p >= 0 else 0) | 1 << t) if ok else 0
                depth = bin(masks[i][t]).count("1") - 1 if ok else 0
            positions[at] = past[i] + depth
            j = (pos - prefix) // page
            if pos >= prefix and j < width and tables[i][j] != NO_PAGE:
                slots[at] = tables[i][j] * page + (pos - prefix) % page
    over = sum(new) - sum(add) + (0 if row_tokens else max(0, sum(add) - n))
    return {"starts": starts, "kv_len": [(past[i] + row_tokens if add[i] else 0) if row_tokens else past[i] + add[i] for i in range(b)],
            "held": kept, "free": free, "positions": positions, "slots": slots, "masks": masks,
            "totals": [sum(add), over, taken, missing]}


def accept(parents, tokens, chosen, n):
    """(path, next) of one tree of n nodes."""
    if n == 0 or parents[0] != -1:
        return [], 0xFFFFFFFF
    path = [0]
    while True:
        want = chosen[path[-1]]
        at = next((j for j in range(path[-1] + 1, n) if parents[j] == path[-1] and tokens[j] == want and want != 0xFFFFFFFF), None)
        if at is None:
            return path, want
        path.append(at)
