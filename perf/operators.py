"""Cases of three operators of a training step, with their plain forms.

* ``distill``: divergence of a student from a teacher that is known on its top token ids, and the gradient of the student's logits;
* ``experts``: routed rows sorted by expert into tiles of the grouped products, brought back with their weights, and both gradients;
* ``embed``: rows of an embedding table times a factor, and the table's gradient by sorted tokens.

``run`` computes them in elementary torch operations where ``own`` is false, and through :mod:`relax_b200.ops` where it is true.
"""
import math

import torch

own = False

TILE = 128                  # rows per tile of the grouped expert products: no tile holds rows of two experts
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one short answer of the smallest vocabulary, every step of which is launches
        {"name": "distill-small", "op": "distill", "rows": 24, "vocab": 1024, "k": 8, "dtype": "fp32", "kl": "reverse_kl", "norm": "tail", "grad": True},
        # a sample's response scored on the teacher's ids for dense rewards: forward only, the log-probs with it
        {"name": "distill-score", "op": "distill", "rows": 512, "vocab": 151936, "k": 64, "dtype": "bf16", "kl": "reverse_kl", "norm": "tail", "grad": False},
        # ragged rows of an odd vocabulary (rows of every alignment), union of two id sets
        {"name": "distill-odd", "op": "distill", "rows": 777, "vocab": 32003, "k": 37, "dtype": "fp32", "kl": "forward_kl", "norm": "norm", "grad": True},
        # a micro-batch in 16-bit logits, symmetric divergence
        {"name": "distill-jsd", "op": "distill", "rows": 2048, "vocab": 151936, "k": 64, "dtype": "bf16", "kl": "jsd", "norm": "tail", "grad": True},
        # one chunk of the fused head: 32-bit logits
        {"name": "distill-chunk", "op": "distill", "rows": 4096, "vocab": 151936, "k": 128, "dtype": "fp32", "kl": "reverse_kl", "norm": "tail", "grad": True},
        # decoding one sequence
        {"name": "experts-one", "op": "experts", "rows": 1, "k": 8, "experts": 128, "hidden": 2048, "dtype": "bf16", "local": 128, "grad": False},
        # decoding a batch where a rank holds a quarter of the experts
        {"name": "experts-decode", "op": "experts", "rows": 96, "k": 8, "experts": 128, "hidden": 2048, "dtype": "bf16", "local": 32, "grad": False},
        # a micro-batch of 128 experts
        {"name": "experts-train", "op": "experts", "rows": 8192, "k": 8, "experts": 128, "hidden": 2048, "dtype": "bf16", "local": 128, "grad": True},
        # ragged rows, few experts, an odd width in 32 bits
        {"name": "experts-odd", "op": "experts", "rows": 3001, "k": 3, "experts": 11, "hidden": 1001, "dtype": "fp32", "local": 11, "grad": True},
        # prompt of the smallest model
        {"name": "embed-small", "op": "embed", "rows": 300, "vocab": 1024, "hidden": 256, "dtype": "fp32", "shards": 1, "scale": 2.0, "grad": True},
        # one of eight shards of a vocabulary, tokens of the others give zeros
        {"name": "embed-shard", "op": "embed", "rows": 8191, "vocab": 151936, "hidden": 5120, "dtype": "bf16", "shards": 8, "scale": 1.0, "grad": True},
        # a micro-batch of 16384 tokens, whole vocabulary
        {"name": "embed-train", "op": "embed", "rows": 16384, "vocab": 151936, "hidden": 4096, "dtype": "bf16", "shards": 1, "scale": 1.0, "grad": True},
    ]


def _span(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("distill", "experts", "embed"))
    if op == "distill":
        vocab, dtype = _span(rng, 500, 152000), rng.choice(("bf16", "bf16", "fp32", "fp16"))
        k = _span(rng, 1, 128)
        kl = rng.choice(("reverse_kl", "forward_kl", "jsd", "low_var_kl"))
        return {"op": op, "rows": _span(rng, 1, min(8192, 600_000_000 // vocab)), "vocab": vocab, "k": k, "dtype": dtype, "kl": kl,
                "norm": rng.choice(("tail", "norm", "trunc")), "grad": rng.random() < 0.7}
    if op == "experts":
        experts = _span(rng, 2, 256)
        hidden = _span(rng, 16, 900) * (8 if rng.random() < 0.8 else 1)
        k = min(experts, rng.randint(1, 8))
        return {"op": op, "rows": _span(rng, 1, min(32768, 130_000_000 // (k * hidden))), "k": k, "experts": experts, "hidden": hidden,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "local": experts if rng.random() < 0.7 else -(-experts // 4),
                "grad": rng.random() < 0.7}
    vocab, shards = _span(rng, 300, 152000), rng.choice((1, 1, 2, 8))
    hidden = _span(rng, 16, 640) * (8 if rng.random() < 0.8 else 1)
    return {"op": op, "rows": _span(rng, 1, 16384), "vocab": max(shards, vocab), "hidden": min(hidden, 600_000_000 // vocab),
            "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "shards": shards, "scale": rng.choice((1.0, 1.0, 45.0)), "grad": rng.random() < 0.7}


# --------------------------------------------------------------------------- inputs


def _capacity(case):
    """Rows of the padded buffer: every expert that has rows ends a tile, at worst each of them a started one."""
    r, e = case["rows"] * case["k"], case["local"]
    n = min(r, e)
    return (n + (r - n) // TILE) * TILE


def _shard(case):
    """Rows of the table here and the id of its first."""
    n = -(-case["vocab"] // case["shards"])
    return n, n * (case["shards"] // 2)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, rows = DTYPES[case["dtype"]], case["rows"]
    draw_n = lambda *s: torch.randn(*s, device="cuda", generator=g)                   # noqa: E731
    draw_u = lambda *s: torch.rand(*s, device="cuda", generator=g)                    # noqa: E731
    s = {}
    if case["op"] == "distill":
        v, k = case["vocab"], case["k"]
        # distinct ids of every row, the teacher's favourites, which the student likes too
        first = (draw_u(rows, 1) * v).long()
        step = 1 + (draw_u(rows, 1) * (max(1, v // k) - 1)).long()
        ids = (first + step * torch.arange(k, device="cuda")) % v
        base = math.log(v) + 4.0 - 6.0 * torch.arange(k, device="cuda") / k
        z = draw_n(rows, v).mul_(2.0)
        z.scatter_(1, ids, base + 1.5 * draw_n(rows, k))
        t = torch.cat([base + draw_n(rows, k), torch.full((rows, 1), math.log(v) + 2.0, device="cuda")], 1)
        s["teacher"] = torch.log_softmax(t.double(), 1)[:, :k].float().contiguous()
        # rows of a union hold different numbers of ids, some none; response masks leave out one token in ten
        held = (draw_u(rows, 1) * 1.5 * k).long().clamp_(max=k)
        ids[torch.arange(k, device="cuda") >= held] = -1
        s["ids"], s["logits"] = ids, z.to(dt)
        s["weight"] = torch.where(draw_u(rows) < 0.1, 0.0, 0.5 + draw_u(rows))
    elif case["op"] == "experts":
        e, k, h, cap = case["experts"], case["k"], case["hidden"], _capacity(case)
        logits = draw_n(rows, e) + draw_n(1, e)                                        # some experts are liked by all
        w, idx = torch.topk(torch.softmax(logits, 1), k, 1)
        s["weights"] = w / w.sum(1, keepdim=True)
        s["expert"] = idx - (0 if case["local"] == e else case["local"])               # ids from here on: others live elsewhere
        s["x"], s["y"] = draw_n(rows, h).to(dt), draw_n(cap, h).to(dt)
        if case["grad"]:
            s["d_sorted"], s["d_out"] = draw_n(cap, h).to(dt), draw_n(rows, h).to(dt)
    else:
        n, start = _shard(case)
        s["tokens"] = (torch.exp(draw_u(rows) * math.log(case["vocab"])).long() * 7919) % case["vocab"]      # few tokens are most of a text
        s["table"], s["start"] = draw_n(n, case["hidden"]).mul_(0.02).to(dt), start
        if case["grad"]:
            s["d_out"] = draw_n(rows, case["hidden"]).to(dt)
    return s


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if case["grad"]:
        for name in ("logits", "x", "y", "weights", "table"):
            if name in s:
                s[name].requires_grad_()
    return s


def work(case):
    rows, size = case["rows"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "distill":
        n, k = rows * case["vocab"], rows * case["k"]
        return {"bytes": n * size * (2 if case["grad"] else 1) + k * (12 if case["grad"] else 16) + rows * (8 if case["grad"] else 4), "flops": n * (10 if case["grad"] else 5)}
    if case["op"] == "experts":
        h, cap, r = case["hidden"], _capacity(case), rows * case["k"]
        there = r * min(1.0, case["local"] / case["experts"])                          # rows of experts that are here, on average
        nbytes = (2 * rows + cap + there) * h * size + r * 16
        flops = 2 * there * h
        if case["grad"]:
            nbytes += (2 * rows + cap + there) * h * size + r * 4
            flops += 4 * there * h
        return {"bytes": nbytes, "flops": flops}
    h, (n, _) = case["hidden"], _shard(case)
    here = rows / case["shards"]
    if not case["grad"]:
        return {"bytes": (here + rows) * h * size + rows * 8, "flops": rows * h}
    return {"bytes": (2 * here + rows + n) * h * size + rows * 8, "flops": 2 * rows * h}


# --------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    return {"distill": _distill, "experts": _experts, "embed": _embed}[case["op"]](state, case)


def _distill(s, case):
    if own:
        from relax_b200 import ops

        if not case["grad"]:
            loss, lp = ops.topk_distill(s["logits"], s["ids"], s["teacher"], kl_type=case["kl"], norm_mode=case["norm"], return_log_probs=True)
            return {"loss": loss, "log_probs": lp}
        loss = ops.topk_distill(s["logits"], s["ids"], s["teacher"], kl_type=case["kl"], norm_mode=case["norm"])
        return {"loss": loss.detach(), "d_logits": torch.autograd.grad(loss, s["logits"], s["weight"])[0]}
    logits, ids, t = s["logits"].detach(), s["ids"], s["teacher"].double()
    there = ids >= 0
    zero = t.new_zeros(())
    z = logits.float()
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    # the student's log-probs of the ids; sums over few ids in 64 bits (the rest's mass is one minus theirs)
    lp = (z.gather(1, ids.clamp_min(0)) - top).double() - torch.log(total)
    p, q = torch.where(there, lp.exp(), zero), torch.where(there, t.exp(), zero)
    least = -math.expm1(-1e-7)                                                         # the rest's mass is no less than this
    if case["kl"] == "low_var_kl":
        r = torch.where(there, lp - t, zero)
        loss = (torch.exp(-r) - 1.0 + r).sum(1)
        c = torch.where(there, 1.0 - torch.exp(-r), zero)
    else:
        if case["norm"] == "norm":
            sp, sq = p.sum(1, keepdim=True), q.sum(1, keepdim=True)
            p, q = torch.where(there, p / sp, zero), torch.where(there, q / sq, zero)
        lp_, lq_ = torch.log(torch.where(there, p, 1.0)), torch.log(torch.where(there, q, 1.0))
        a = 0.5
        lm_ = torch.log(torch.where(there, (1.0 - a) * p + a * q, 1.0))

        def term(p, q, lp, lq, lm):
            if case["kl"] == "reverse_kl":
                return p * (lp - lq)
            if case["kl"] == "forward_kl":
                return q * (lq - lp)
            return (1.0 - a) * p * (lp - lm) + a * q * (lq - lm)

        def slope(p, q, lp, lq, lm):                                                   # d term / d p, times p
            if case["kl"] == "reverse_kl":
                return p * (lp - lq + 1.0)
            if case["kl"] == "forward_kl":
                return -q
            return (1.0 - a) * p * (lp - lm)

        loss = term(p, q, lp_, lq_, lm_).sum(1)
        c = slope(p, q, lp_, lq_, lm_)
        if case["norm"] == "norm":
            c = c - p * c.sum(1, keepdim=True)
        if case["norm"] == "tail":
            free = 1.0 - p.sum(1)
            pr, qr = free.clamp_min(least), (1.0 - q.sum(1)).clamp_min(least)
            rest = (pr, qr, torch.log(pr), torch.log(qr), torch.log((1.0 - a) * pr + a * qr))
            loss = loss + term(*rest)
            c = c - p * torch.where(free >= least, slope(*rest) / pr, zero)[:, None]
    if not case["grad"]:
        return {"loss": loss.float(), "log_probs": torch.where(there, lp, -math.inf).float()}
    c = (c * s["weight"].double()[:, None]).float()
    d = e * (-c.sum(1, keepdim=True) / total.float())
    d.scatter_add_(1, ids.clamp_min(0), c)
    return {"loss": loss.float(), "d_logits": d.to(logits.dtype)}


def _experts(s, case):
    if own:
        from relax_b200 import ops

        rows = ops.expert_layout(s["expert"], case["local"])
        srt = ops.expert_dispatch(s["x"], rows)
        out = ops.expert_combine(s["y"], s["weights"], rows)
        found = {"place": rows.dest, "tiles": rows.tile_expert, "bounds": rows.expert_rows}
        if not case["grad"]:
            return {**found, "sorted": srt, "out": out}
        d = torch.autograd.grad([srt, out], [s["x"], s["y"], s["weights"]], [s["d_sorted"], s["d_out"]])
        return {**found, "sorted": srt.detach(), "out": out.detach(), "d_x": d[0], "d_y": d[1], "d_weights": d[2]}
    x, y, w, e = s["x"].detach(), s["y"].detach(), s["weights"].detach(), s["expert"].reshape(-1)
    k, n, cap, dev = case["k"], case["local"], _capacity(case), x.device
    here = (e >= 0) & (e < n)
    key = torch.where(here, e, n)
    count = torch.zeros(n + 1, dtype=torch.int64, device=dev).index_add_(0, key, torch.ones_like(key))
    padded = (count[:n] + TILE - 1) // TILE * TILE
    ends = padded.cumsum(0)
    order = torch.argsort(key, stable=True)
    before = torch.cat([count.new_zeros(1), count.cumsum(0)])[key[order]]              # sorted rows of the experts in front
    place = torch.cat([ends - padded, ends[-1:]])[key[order]] + torch.arange(e.numel(), device=dev) - before
    dest = torch.empty_like(key)
    dest[order] = torch.where(here[order], place, -1)
    start = torch.arange(cap // TILE, device=dev) * TILE
    tiles = torch.searchsorted(ends, start, right=True)
    tiles = torch.where(tiles < n, tiles, -1).int()
    bounds = torch.cat([ends.new_zeros(1), ends]).int()
    spare = torch.where(dest < 0, cap, dest)                                           # a row behind the buffer for rows of other ranks
    srt = x.new_zeros(cap + 1, x.shape[1]).index_copy_(0, spare, torch.where(here[:, None], x.repeat_interleave(k, 0), 0))[:cap]
    rows = torch.where(here[:, None], y[dest.clamp_min(0)], 0).float()
    wf = w.float().reshape(-1, 1)
    out = (rows * wf).view(-1, k, x.shape[1]).sum(1).to(x.dtype)
    found = {"place": dest.view(-1, k).int(), "tiles": tiles, "bounds": bounds}
    if not case["grad"]:
        return {**found, "sorted": srt, "out": out}
    d_rows = torch.where(here[:, None], s["d_sorted"][dest.clamp_min(0)], 0).float()
    d_x = d_rows.view(-1, k, x.shape[1]).sum(1).to(x.dtype)
    up = s["d_out"].float().repeat_interleave(k, 0)
    d_y = torch.zeros(cap + 1, x.shape[1], device=dev).index_copy_(0, spare, up * wf)[:cap].to(y.dtype)
    return {**found, "sorted": srt, "out": out, "d_x": d_x, "d_y": d_y, "d_weights": (rows * up).sum(1).view(-1, k)}


def _embed(s, case):
    if own:
        from relax_b200 import ops

        out = ops.embedding(s["tokens"], s["table"], scale=case["scale"], vocab_start=s["start"])
        if not case["grad"]:
            return {"out": out}
        return {"out": out.detach(), "d_table": torch.autograd.grad(out, s["table"], s["d_out"])[0]}
    table = s["table"].detach()
    at = s["tokens"] - s["start"]
    here = (at >= 0) & (at < table.shape[0])
    at = torch.where(here, at, 0)
    out = (table[at].float() * torch.where(here, case["scale"], 0.0)[:, None]).to(table.dtype)
    if not case["grad"]:
        return {"out": out}
    up = torch.where(here[:, None], s["d_out"].float(), 0.0)
    d = torch.zeros(table.shape, device=table.device).index_add_(0, at, up)
    return {"out": out, "d_table": (d * case["scale"]).to(table.dtype)}


# --------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "distill":
        return _exact_distill(s, case)
    if case["op"] == "experts":
        return _exact_experts(s, case)
    n, h = s["table"].shape
    at = s["tokens"] - s["start"]
    here = ((at >= 0) & (at < n)).nonzero()[:, 0]
    out = torch.zeros(case["rows"], h, dtype=torch.float64, device="cuda")
    out[here] = s["table"][at[here]].double() * case["scale"]
    if not case["grad"]:
        return {"out": out}
    d = torch.zeros(n, h, dtype=torch.float64, device="cuda")
    d.index_put_((at[here],), s["d_out"][here].double() * case["scale"], accumulate=True)
    return {"out": out, "d_table": d}


def _exact_distill(s, case):
    """The divergence as written, differentiated by autograd."""
    z = s["logits"].double().requires_grad_(case["grad"])
    away = s["ids"] < 0
    lp = (z - torch.logsumexp(z, 1, keepdim=True)).gather(1, s["ids"].clamp_min(0))
    found = lp.masked_fill(away, -math.inf)
    lq = s["teacher"].double()
    if case["kl"] == "low_var_kl":
        r = lp - lq
        loss = (torch.exp(-r) - 1 + r).masked_fill(away, 0.0).sum(1)
    else:
        big = -1e30                                                                    # (finite, so that absent ids have gradients of zero)
        lp, lq = lp.masked_fill(away, big), lq.masked_fill(away, big)
        if case["norm"] == "norm":
            lp, lq = torch.log_softmax(lp, 1), torch.log_softmax(lq, 1)
            keep = ~away
        elif case["norm"] == "tail":
            rest = lambda l: torch.log(-torch.expm1(torch.logsumexp(l, 1, keepdim=True).clamp(max=-1e-7)))      # noqa: E731
            lp, lq = torch.cat([lp, rest(lp)], 1), torch.cat([lq, rest(lq)], 1)
            keep = torch.cat([~away, torch.ones_like(away[:, :1])], 1)
        else:
            keep = ~away
        kl = lambda p, q: (p.exp() * (p - q)).masked_fill(~keep, 0.0).sum(1)           # noqa: E731
        mid = torch.logaddexp(lp, lq) - math.log(2.0)
        loss = {"reverse_kl": lambda: kl(lp, lq), "forward_kl": lambda: kl(lq, lp), "jsd": lambda: 0.5 * kl(lp, mid) + 0.5 * kl(lq, mid)}[case["kl"]]()
    if not case["grad"]:
        return {"loss": loss, "log_probs": found}
    d = torch.autograd.grad(loss, z, s["weight"].double())[0]
    return {"loss": loss.detach(), "d_logits": d}


def _exact_experts(s, case):
    e, k, cap, h = s["expert"].cpu(), case["k"], _capacity(case), case["hidden"]
    dest = torch.full((e.numel(),), -1, dtype=torch.int64)
    at = 0
    for expert in range(case["local"]):
        mine = (e.reshape(-1) == expert).nonzero()[:, 0]
        dest[mine] = at + torch.arange(mine.numel())
        at += -(-mine.numel() // TILE) * TILE
    dest = dest.cuda()
    flat = (dest >= 0).nonzero()[:, 0]
    place, token = dest[flat], flat // k
    zeros = lambda n: torch.zeros(n, h, dtype=torch.float64, device="cuda")            # noqa: E731
    w = s["weights"].double().reshape(-1)[flat][:, None]
    x, y = s["x"].double(), s["y"].double()
    srt, out = zeros(cap), zeros(case["rows"])
    srt[place] = x[token]
    out.index_add_(0, token, y[place] * w)
    found = {"place": None, "tiles": None, "bounds": None, "sorted": srt, "out": out}
    if not case["grad"]:
        return found
    d_x, d_y, d_w = zeros(case["rows"]), zeros(cap), torch.zeros(e.numel(), dtype=torch.float64, device="cuda")
    d_x.index_add_(0, token, s["d_sorted"].double()[place])
    up = s["d_out"].double()[token]
    d_y[place] = up * w
    d_w[flat] = (up * y[place]).sum(1)
    return {**found, "d_x": d_x, "d_y": d_y, "d_weights": d_w.view(-1, k)}
