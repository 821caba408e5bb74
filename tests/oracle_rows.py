"""Plain statements in 64 bits of the operators that move rows by key and of the distillation divergence, one row at a time."""
import math

import torch


def layout(ids, experts, align):
    """``(dest, source, tiles, bounds)`` as lists, by walking over the experts."""
    flat = [int(e) for row in ids.tolist() for e in row]
    n = len(flat)
    some = min(n, experts)
    cap = n if align == 1 else (some + (n - some) // align) * align
    dest, source, tiles, bounds, at = [-1] * n, [-1] * cap, [], [0], 0
    for e in range(experts):
        mine = [i for i, x in enumerate(flat) if x == e]
        for j, i in enumerate(mine):
            dest[i], source[at + j] = at + j, i
        used = -(-len(mine) // align)
        tiles += [e] * used
        at += used * align
        bounds.append(at)
    tiles += [-1] * (cap // align - len(tiles))
    return dest, source, tiles, bounds


def dispatch(x, source, k):
    out = torch.zeros(len(source), x.shape[1], dtype=torch.float64)
    for r, s in enumerate(source):
        if s >= 0:
            out[r] = x[s // k].double()
    return out


def combine(y, w, dest, k):
    """``(sum, sum of absolute terms)`` per row."""
    T = len(dest) // k
    out, size = (torch.zeros(T, y.shape[1], dtype=torch.float64) for _ in range(2))
    for i, d in enumerate(dest):
        if d >= 0:
            v = y[d].double() * (1.0 if w is None else float(w.reshape(-1)[i]))
            out[i // k] += v
            size[i // k] += v.abs()
    return out, size


def embedding_grad(tokens, dy, rows, start, scale):
    g, size = (torch.zeros(rows, dy.shape[1], dtype=torch.float64) for _ in range(2))
    for i, t in enumerate(tokens.reshape(-1).tolist()):
        if 0 <= t - start < rows:
            g[t - start] += dy[i].double() * scale
            size[t - start] += dy[i].double().abs() * abs(scale)
    return g, size


LEAST = -1e-7       # the log of the most mass that the ids may hold


def distill_row(z, ids, teacher, kl, alpha, norm, temperature, clamp):
    """The divergence of one row from whole logits ``z`` (64 bits, may require gradients), and a measure of its terms."""
    lp = torch.log_softmax(z / temperature, 0)
    cols = [i for i, v in enumerate(ids.tolist()) if 0 <= v < z.shape[0]]
    s = lp[ids[cols]] if cols else lp[:0]
    t = teacher[cols].double()
    if clamp is not None:
        s, t = s.clamp_min(clamp), t.clamp_min(clamp)
    if kl == "low_var_kl":
        return sum((torch.exp(t[i] - s[i]) - 1 + s[i] - t[i] for i in range(len(cols))), z.sum() * 0), float((torch.exp(t - s) + 1 + (t - s).abs()).sum())
    p, q = list(s.exp()), list(t.exp())
    if norm == "norm" and cols:
        sp, sq = sum(p), sum(q)
        p, q = [x / sp for x in p], [x / sq for x in q]
    if norm == "tail":
        least = -math.expm1(LEAST)
        rp, rq = (1 - sum(x, torch.zeros((), dtype=torch.float64)) for x in (p, q))
        p, q = p + [rp if float(rp) >= least else torch.tensor(least, dtype=torch.float64)], q + [rq if float(rq) >= least else torch.tensor(least, dtype=torch.float64)]
    a = {"reverse_kl": 0.0, "forward_kl": 1.0}.get(kl, alpha)
    total, size = z.sum() * 0, 1.0
    for x, y in zip(p, q):
        m = (1 - a) * x + a * y
        if a < 1 and float(x) > 0:
            total = total + (1 - a) * x * (torch.log(x) - torch.log(y if a == 0 else m))
        if a > 0 and float(y) > 0:
            total = total + a * y * (torch.log(y) - torch.log(x if a == 1 else m))
        if float(x) > 0 and float(y) > 0:
            # the divergence's term and its slope's: what a relative error of the masses is multiplied by
            size += (float(x) + float(y)) * (abs(math.log(float(x)) - math.log(float(y))) + 2.0)
    if norm == "tail":
        size *= 1.0 + float(q[-1]) / float(p[-1]) + abs(math.log(float(q[-1])) - math.log(float(p[-1])))
    return total, size


def distill(z, ids, teacher, weight, kl="reverse_kl", alpha=0.5, norm="tail", temperature=1.0, clamp=None):
    """``(loss, d logits of sum(weight * loss), size)`` with everything in 64 bits on the CPU."""
    z = z.detach().cpu().double().requires_grad_()
    ids, teacher, weight = ids.cpu(), teacher.cpu(), weight.cpu().double()
    got = [distill_row(z[r], ids[r], teacher[r], kl, alpha, norm, temperature, clamp) for r in range(z.shape[0])]
    loss = torch.stack([g[0] for g in got]) if got else z.sum(1)
    (d,) = torch.autograd.grad((loss * weight).sum(), z)
    return loss.detach(), d, torch.tensor([g[1] for g in got], dtype=torch.float64)
