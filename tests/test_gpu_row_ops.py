"""sm_100a kernels of rows sorted by expert and back, the embedding with its gradient and the distillation divergence, against plain statements in 64
bits.  Tolerances count roundings: half a step of the result's type (eps / 2) and 2^-24 per 32-bit operation."""
import math

import pytest
import torch

import oracle_rows as O
from relax_b200 import ops

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _half_step(t):
    return torch.finfo(t).eps / 2


def _within(got, want, tol, what=""):
    got = got.detach().double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() - tol).max()):.3e} over"


# --------------------------------------------------------------------------- experts' rows


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("T,k,E,align", [(0, 2, 4, 128), (1, 1, 1, 128), (1, 8, 128, 128), (96, 8, 32, 128), (513, 3, 11, 128), (5000, 2, 300, 128), (2500, 8, 256, 1),
                                         (1700, 3, 2048, 16), (7, 40, 60, 128), (9001, 1, 5, 1), (16384, 1, 33, 128), (16385, 1, 2048, 128), (30000, 3, 64, 128)])
def test_layout(T, k, E, align, wide):
    g = torch.Generator().manual_seed(T + k)
    ids = (torch.randn(T, k, generator=g) * E * 0.6).long()              # half of them elsewhere, experts of very different load
    rows = ops.expert_layout((ids if wide else ids.int()).cuda(), E, align)
    dest, source, tiles, bounds = O.layout(ids, E, align)
    assert rows.dest.shape == (T, k) and rows.dest.reshape(-1).tolist() == dest
    assert rows.source.tolist() == source and rows.expert_rows.tolist() == bounds
    assert rows.tile_expert is None if align == 1 else rows.tile_expert.tolist() == tiles


@pytest.mark.parametrize("pattern", ["one expert", "all elsewhere", "descending"])
def test_layout_of_lopsided_rows(pattern):
    n = 6000
    ids = {"one expert": torch.full((n, 1), 3), "all elsewhere": torch.full((n, 1), -1), "descending": torch.arange(n - 1, -1, -1)[:, None] // 60}[pattern]
    rows = ops.expert_layout(ids.cuda(), 100, 128)
    dest, source, tiles, bounds = O.layout(ids, 100, 128)
    assert rows.dest.reshape(-1).tolist() == dest and rows.source.tolist() == source
    assert rows.tile_expert.tolist() == tiles and rows.expert_rows.tolist() == bounds


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (1, 8, 128, 2048), (70, 2, 9, 1), (333, 3, 11, 1001), (260, 8, 16, 264), (50, 37, 40, 520)])
def test_dispatch_and_combine(T, k, E, H, dtype):
    dt, g = DT[dtype], _gen(T + H)
    ids = torch.randint(-1, E + 1, (T, k), device="cuda", generator=g)
    rows = ops.expert_layout(ids, E)
    dest, source, _, _ = O.layout(ids.cpu(), E, 128)
    cap = len(source)
    x = torch.randn(T, H + 8, device="cuda", generator=g).to(dt)[:, :H].requires_grad_()               # rows apart from one another
    y = torch.randn(cap, H, device="cuda", generator=g).to(dt)
    pad = torch.tensor(source) < 0
    y[pad.cuda()] = float("nan")                                                                       # padding is not looked at
    y.requires_grad_()
    w = torch.rand(T, k, device="cuda", generator=g)
    w[ids < 0] = float("inf")                                                                          # nor are weights of rows elsewhere
    w.requires_grad_()
    srt, out = ops.expert_dispatch(x, rows), ops.expert_combine(y, w, rows)
    assert torch.equal(srt.detach().double().cpu(), O.dispatch(x.detach().cpu(), source, k))
    yc, wc = y.detach().cpu(), w.detach().cpu()
    want, size = O.combine(yc, wc, dest, k)
    half = _half_step(dt)
    _within(out, want, half * want.abs() + (1 + half) * (k + 1) * F * size + 2.0 ** -25, "combine")
    _within(ops.expert_combine(y, w, rows, torch.float32), want, (k + 1) * F * size, "combine in fp32")
    plain, psize = O.combine(yc, None, dest, k)
    _within(ops.expert_combine(y, None, rows), plain, half * plain.abs() + (1 + half) * (k + 1) * F * psize + 2.0 ** -25, "plain sum")

    d_s, d_o = torch.randn(cap, H, device="cuda", generator=g).to(dt), torch.randn(T, H, device="cuda", generator=g).to(dt)
    d_x, d_y, d_w = torch.autograd.grad([srt, out], [x, y, w], [d_s, d_o])
    want, size = O.combine(d_s.cpu(), None, dest, k)
    _within(d_x, want, half * want.abs() + (1 + half) * (k + 1) * F * size + 2.0 ** -25, "d x")
    doc = d_o.cpu().double()
    want_y, want_w, size_w = torch.zeros(cap, H, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
    for i, d in enumerate(dest):
        if d >= 0:
            want_y[d] = doc[i // k] * float(wc.reshape(-1)[i])
            terms = doc[i // k] * yc[d].double()
            want_w[i], size_w[i] = terms.sum(), terms.abs().sum()
    _within(d_y, want_y, (half + 2 * F) * want_y.abs() + 2.0 ** -25, "d y")
    _within(d_w.reshape(-1), want_w, (H / 32 + 8) * F * size_w, "d weights")      # a lane sums H / 32 terms, five more additions join the lanes


@pytest.mark.parametrize("T,k,E,H,align,dtype", [(8193, 3, 40, 1552, 128, "bf16"), (6200, 33, 300, 2048, 4, "fp16"), (26000, 2, 7, 520, 1, "bf16"), (3000, 5, 64, 2100, 128, "fp32")])
def test_dispatch_of_many_rows(T, k, E, H, align, dtype):
    """Rows that are read once and put down at all their places: every row of the buffer is written, padding with zeros."""
    g = _gen(31)
    ids = torch.randint(-1, E + 1, (T, k), device="cuda", generator=g)      # (some live elsewhere, some come twice)
    x = torch.randn(T, H + 8, device="cuda", generator=g).to(DT[dtype])[:, 8 * (k % 2): 8 * (k % 2) + H]
    rows = ops.expert_layout(ids, E, align)
    out = ops.expert_dispatch(x, rows)
    s = rows.source.long()
    want = torch.where((s >= 0)[:, None], x[torch.div(s.clamp_min(0), k, rounding_mode="floor")], torch.zeros((), device="cuda", dtype=DT[dtype]))
    assert torch.equal(out, want)


def test_rows_again_give_the_same_bits_and_may_be_captured():
    g = _gen(5)
    ids = torch.randint(0, 16, (700, 4), device="cuda", generator=g)
    x = torch.randn(700, 256, device="cuda", generator=g).bfloat16()
    w = torch.rand(700, 4, device="cuda", generator=g)
    tok = torch.randint(0, 50, (5000,), device="cuda", generator=g)
    table = torch.randn(64, 256, device="cuda", generator=g).bfloat16()
    dy = torch.randn(5000, 256, device="cuda", generator=g).bfloat16()

    def all_of_them():
        rows = ops.expert_layout(ids, 16)
        y = ops.expert_dispatch(x, rows)
        t = table.detach().requires_grad_()
        d = torch.autograd.grad(ops.embedding(tok, t, 2.0), t, dy)[0]
        return [rows.dest, rows.source, y, ops.expert_combine(y, w, rows), d]

    first = [t.clone() for t in all_of_them()]
    assert all(torch.equal(a, b) for a, b in zip(first, all_of_them()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of_them()
        again = all_of_them()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_of_them()
    ids.copy_(torch.randint(0, 16, (700, 4), device="cuda", generator=g))
    tok.copy_(torch.randint(0, 50, (5000,), device="cuda", generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip([t.clone() for t in held], all_of_them()))


def test_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    rows = ops.expert_layout(ids, 3)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.expert_dispatch(torch.zeros(4, 8, device="cuda", dtype=torch.float64), rows)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.embedding(ids[:, 0], torch.zeros(4, 8, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="is on"):
        ops.embedding(ids[:, 0].cpu(), torch.zeros(4, 8, device="cuda"))
    with pytest.raises(ValueError, match="is on"):
        ops.expert_dispatch(torch.zeros(4, 8, device="cuda"), ops.expert_layout(ids.cpu(), 3))
    with pytest.raises(ValueError, match="is on"):
        ops.topk_distill(torch.zeros(4, 8, device="cuda"), ids.cpu(), torch.zeros(4, 2, device="cuda"))
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.topk_distill(torch.zeros(4, 8, device="cuda", dtype=torch.float64), ids, torch.zeros(4, 2, device="cuda"))
    with pytest.raises(ValueError, match="float32"):
        ops.expert_combine(torch.zeros(rows.source.numel(), 8, device="cuda"), None, rows, torch.bfloat16)
    with pytest.raises(TypeError, match="bf16"):
        ops.fused_lm_head_topk_distill(torch.zeros(4, 8, device="cuda"), torch.zeros(16, 8, device="cuda"), ids, torch.zeros(4, 2, device="cuda"))
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.fused_lm_head_topk_distill(torch.zeros(4, 8, device="cuda").bfloat16(), torch.zeros(15, 8, device="cuda").bfloat16(), ids,
                                       torch.zeros(4, 2, device="cuda"))


# --------------------------------------------------------------------------- embedding


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,V,H,start,scale,tokens", [
    (0, 16, 8, 0, 1.0, "few"), (1, 1, 1, 0, 1.0, "few"), (33, 7, 3, 0, 45.0, "few"), (700, 1000, 264, 0, 1.0, "few"), (9000, 151936, 40, 0, 1.0, "zipf"),
    (5000, 2000, 136, 4000, 2.0, "zipf"), (5000, 300, 72, 0, 1.0, "one"), (8300, 2500, 11, 0, 1.0, "runs"), (64, 1 << 20, 8, 0, 1.0, "zipf")])
def test_embedding(n, V, H, start, scale, tokens, dtype):
    dt, g = DT[dtype], _gen(n + H)
    u = torch.rand(n, device="cuda", generator=g)
    ids = {"few": (u * (V + 2)).long() - 1, "zipf": torch.exp(u * math.log(V + start)).long() - 1, "one": torch.full((n,), V - 1, device="cuda"),
           "runs": torch.arange(n, device="cuda") // 32 % V}[tokens]
    table = torch.randn(V, H, device="cuda", generator=g).to(dt).requires_grad_()
    out = ops.embedding(ids, table, scale, start)
    at = (ids - start).cpu()
    here = (at >= 0) & (at < V)
    want = torch.where(here[:, None], table.detach().cpu().double()[at.clamp(0, V - 1)] * scale, torch.zeros((), dtype=torch.float64))
    half = _half_step(dt)
    _within(out, want, 0.0 if scale == 1.0 else (half + 2 * F) * want.abs(), "rows")
    dy = torch.randn(n, H, device="cuda", generator=g).to(dt)
    (d,) = torch.autograd.grad(out, table, dy)
    here_at = at[here]
    c = torch.zeros(V, dtype=torch.float64).index_add_(0, here_at, torch.ones(here_at.numel(), dtype=torch.float64))
    up = dy.cpu().double()[here] * scale
    want = torch.zeros(V, H, dtype=torch.float64).index_add_(0, here_at, up)
    size = torch.zeros(V, H, dtype=torch.float64).index_add_(0, here_at, up.abs())
    sums = (c[:, None] + 2) * F * size
    assert d.dtype == dt
    _within(d, want, half * want.abs() + (1 + half) * sums + 2.0 ** -25, "gradient")
    # into the optimizer's buffer: one more addition
    table.main_grad = torch.randn(V, H, device="cuda", generator=g)
    before = table.main_grad.cpu().double()
    ops.embedding(ids, table, scale, start).backward(dy)
    assert table.grad is None
    _within(table.main_grad, before + want, sums + F * (before.abs() + want.abs() + sums), "main_grad")
    untouched = c == 0
    assert torch.equal(table.main_grad.cpu().double()[untouched], before[untouched])


def test_embedding_of_odd_views():
    g = _gen(1)
    table = torch.randn(50, 24, device="cuda", generator=g).bfloat16()[:, 3:20]                 # rows that begin anywhere
    ids = torch.randint(0, 50, (4, 9), device="cuda", generator=g, dtype=torch.int32)
    assert torch.equal(ops.embedding(ids, table), table[ids.long()])
    assert torch.equal(ops.embedding(ids.t(), table), table[ids.t().long()])
    leaf = table.contiguous().requires_grad_()
    dy = torch.randn(4, 17, device="cuda", generator=g).bfloat16()[:, None].expand(4, 9, 17)      # a broadcast gradient
    (d,) = torch.autograd.grad(ops.embedding(ids, leaf), leaf, dy)
    want, size = O.embedding_grad(ids.cpu(), dy.reshape(-1, 17).cpu(), 50, 0, 1.0)
    _within(d, want, 2.0 ** -8 * want.abs() + 40 * F * size, "gradient")


@pytest.mark.parametrize("n", [1, 31, 1024, 1025, 4097, 16384, 16385, 40000])
@pytest.mark.parametrize("V", [3, 1023, 1024, 151936, (1 << 18) - 1, 1 << 18, 1 << 20, 3000001])
def test_embedding_sort(n, V):
    """Every way of sorting: one launch or several, one pass or more, keys up to and beyond a power of two, runs that cross chunks."""
    g = _gen(n + V)
    ids = torch.randint(-1, V + 1, (n,), device="cuda", generator=g)
    ids[: n // 2] = ids[: n // 2] % 40                       # half of the tokens share few rows
    ids[-1] = V - 1
    table = torch.zeros(V, 4, device="cuda").requires_grad_()
    dy = torch.randint(-8, 9, (n, 4), device="cuda", generator=g).float()        # whole numbers: sums are exact in any order
    (d,) = torch.autograd.grad(ops.embedding(ids, table), table, dy)
    ok = (ids >= 0) & (ids < V)
    assert torch.equal(d, torch.zeros(V, 4, device="cuda").index_add_(0, ids[ok], dy[ok]))


# --------------------------------------------------------------------------- distillation


def _case(R, V, K, dtype, seed, spread=3.0):
    g = _gen(seed)
    z = (spread * torch.randn(R, V, device="cuda", generator=g)).to(DT[dtype])
    ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:K] for _ in range(R)]) if R else torch.zeros(0, K, dtype=torch.int64, device="cuda")
    t = torch.log_softmax(2.0 * torch.randn(R, K + 1, device="cuda", generator=g), 1)[:, :K].contiguous()
    w = 0.5 + torch.rand(R, device="cuda", generator=g)
    return z, ids, t, w


def _check(z, ids, t, w, **kw):
    """Loss and gradient against 64 bits.  With A the widest exponent of a row: the exponentials are off by 2^-22 (the instruction) and A 2^-23
    (their arguments, the rounded factor log2(e) / T), their sum by (V / 2048 + 40) 2^-24 more; every mass and log-prob is off by at most a
    small multiple of that, and the divergence and its slopes by as much times their terms (`size`)."""
    temperature = kw.get("temperature", 1.0)
    zl = z.detach().requires_grad_()
    loss = ops.topk_distill(zl, ids, t, kw.get("kl", "reverse_kl"), kw.get("alpha", 0.5), kw.get("norm", "tail"), temperature, kw.get("clamp"))
    (d,) = torch.autograd.grad(loss, zl, w)
    want, d_want, size = O.distill(z, ids, t, w, **kw)
    A = (z.double().cpu().amax(1) - z.double().cpu().amin(1)) / temperature * 1.5 + z.double().cpu().abs().amax(1) / temperature
    off = 4 * (2.0 ** -22 + (2 * A + z.shape[1] / 2048 + 40) * F)
    _within(loss, want, off * size + F * want.abs(), f"loss {kw}")
    p = torch.softmax(z.double().cpu() / temperature, 1)
    at = torch.zeros_like(p)
    idc = ids.cpu()
    ok = (idc >= 0) & (idc < z.shape[1])
    rows = torch.arange(z.shape[0])[:, None].expand_as(idc)
    at[rows[ok], idc[ok]] = 1.0
    g = w.cpu().double()[:, None] / temperature
    half = _half_step(d.dtype)
    tol = g * (off * size)[:, None] * (p + at)
    _within(d, d_want, half * d_want.abs() + (1 + half) * tol + (2.0 ** -25 if d.dtype == torch.float16 else 1e-37), f"gradient {kw}")
    return loss, d


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,V,K", [(1, 1, 1), (1, 7, 3), (5, 1000, 8), (3, 4099, 64), (6, 33001, 17), (150, 515, 128), (2, 151936, 64), (0, 100, 4), (4, 16, 0)])
def test_distill(R, V, K, dtype):
    z, ids, t, w = _case(R, V, K, dtype, R + V)
    if R > 2 and K > 2:
        ids[0, K // 2:] = -1
        ids[1] = V + 5                                          # nothing of this row is known
        w[2] = 0.0                                              # nor asked of this one
    loss, d = _check(z, ids, t, w)
    if R > 2 and K > 2:
        assert float(loss[1]) == 0.0 and not d[1].any() and not d[2].any()


@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd", "low_var_kl"])
@pytest.mark.parametrize("norm", ["tail", "norm", "trunc"])
@pytest.mark.parametrize("clamp,temperature", [(None, 1.0), (-6.0, 0.7), (None, 3.0)])
def test_distill_divergences(kl, norm, clamp, temperature):
    z, ids, t, w = _case(9, 2050, 33, "fp32", 4, 2.0)
    z[torch.arange(9, device="cuda")[:, None], ids[:, :6]] += 9.0           # rows whose ids hold most of the mass
    ids[3, 5:] = -1
    ids[4] = -1
    _check(z, ids, t, w, kl=kl, alpha=0.3, norm=norm, clamp=clamp, temperature=temperature)


def test_distill_where_the_ids_hold_everything():
    """1 - sum P has no digits left in 32 bits; the mass outside is summed by itself, down to its floor."""
    for lift in (8.0, 14.0, 17.0, 30.0):
        z, ids, t, w = _case(4, 3001, 5, "fp32", 6, 1.0)
        z[torch.arange(4, device="cuda")[:, None], ids] += lift
        for kl in ("reverse_kl", "forward_kl", "jsd"):
            _check(z, ids, t, w, kl=kl)


def test_distill_ids_twice_and_views():
    z, ids, t, w = _case(5, 700, 12, "bf16", 8)
    ids[:, 7] = ids[:, 2]
    ids[1, :] = ids[1, 0]
    t = t - 2.0                                                  # (so that equal ids together stay below one)
    z2 = torch.zeros(5, 720, device="cuda", dtype=torch.bfloat16)
    z2[:, 5:705] = z
    for norm in ("tail", "norm", "trunc"):
        a = _check(z, ids, t, w, norm=norm)
        b = _check(z2[:, 5:705], ids, t, w, norm=norm)           # rows that begin anywhere
        assert torch.allclose(a[0], b[0], rtol=1e-5, atol=1e-6)
    c = ops.topk_distill(z.t().contiguous().t(), ids, t)         # columns first
    assert torch.equal(c, ops.topk_distill(z, ids, t))


def test_distill_infinities():
    z, ids, t, w = _case(4, 600, 6, "fp32", 12)
    z[:, 300:] = -math.inf                                       # tokens that the student cannot give
    ids[0, 0] = 400
    ids[1:] = ids[1:] % 300
    t[1, 2] = -math.inf
    loss = ops.topk_distill(z, ids, t)
    ref = ops.topk_distill(z.cpu(), ids.cpu(), t.cpu())
    assert torch.isinf(loss[1]) and torch.allclose(loss[[0, 2, 3]].cpu(), ref[[0, 2, 3]], rtol=1e-4, atol=1e-5)
    z[3, 17] = math.nan
    out = ops.topk_distill(z, ids, t, "forward_kl")
    assert torch.isnan(out[3]) and torch.isinf(out[0]) and torch.isfinite(out[[1, 2]]).all()


@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.5, 3.0])      # (what 32 bits leave of log2(e) / T is below zero at the first, third and last)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_distill_masks_at_any_temperature(dtype, temperature):
    """Tokens masked with -inf have no mass and no gradient; the others are as if they stood alone."""
    z, ids, t, w = _case(6, 1500, 9, dtype, 16)
    want, d_want = _check(z, ids, t, w, kl="jsd", temperature=temperature)
    masked = torch.nn.functional.pad(z, (0, 700), value=-math.inf).requires_grad_()
    loss = ops.topk_distill(masked, ids, t, "jsd", temperature=temperature)
    (d,) = torch.autograd.grad(loss, masked, w)
    assert bool((d[:, 1500:] == 0).all())
    assert torch.allclose(loss, want, rtol=1e-5, atol=1e-6)      # (other parts of a row: other orders of the sum, 2e-6 of it)
    assert torch.allclose(d[:, :1500].float(), d_want.float(), rtol=4 * _half_step(d.dtype) + 1e-5, atol=1e-6)


@pytest.mark.parametrize("at", [0, 1, 800, 1002])
def test_distill_nan_between_masks(at):
    """A NaN is not lost in a row of nothing but the type's lowest value, nor is a row of NaN."""
    z, ids, t, w = _case(3, 1003, 4, "fp32", 17)
    ids[:] = torch.tensor([5, 6, 7, 9], device="cuda")
    z[0] = torch.finfo(torch.float32).min
    z[0, at] = math.nan
    z[1] = math.nan
    loss, lp = ops.topk_distill(z, ids, t, return_log_probs=True)
    assert torch.isnan(loss[:2]).all() and torch.isnan(lp[:2]).all() and torch.isfinite(loss[2])


@pytest.mark.parametrize("temperature", [0.3, 1.0, 5.03])
@pytest.mark.parametrize("mask", [-1e5, -3e6, -1e9, -2e10, -1e30, -3.3e38])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_distill_masks_of_any_value(dtype, mask, temperature):
    """Masked tokens have no mass beside others, wherever they lie and however many follow one another; rows of nothing else are uniform."""
    z, ids, t, w = _case(5, 20003, 12, dtype, 23)
    z[0] = mask
    z[1, 40:] = mask
    z[2, ::2] = mask
    z[3, :19000] = mask
    ids[1] = torch.arange(4, 28, 2, device="cuda")
    ids[3] += 100      # (masked ones among them)
    ids.remainder_(20003)
    for kl, norm in (("forward_kl", "trunc"), ("jsd", "tail")):
        zl = z.detach().requires_grad_()
        loss = ops.topk_distill(zl, ids, t, kl, norm_mode=norm, temperature=temperature, log_prob_min_clamp=-30.0)
        (d,) = torch.autograd.grad(loss, zl, w)
        want, d_want, _ = O.distill(z, ids, t, w, kl, 0.5, norm, temperature, -30.0)
        # far rows: logits of one value, whose 64-bit exponents are alike but for 2^-53 of 1e10; others as in the tests above
        assert torch.allclose(loss.double().cpu(), want, rtol=3e-5, atol=1e-5)
        top = d_want.abs().amax(1, keepdim=True)
        assert bool(((d.double().cpu() - d_want).abs() <= (2 * _half_step(d.dtype) + 1e-4) * d_want.abs() + 1e-6 * top + 1e-30).all())


def test_distill_far_logits_are_told_apart():
    """Rows whose logits lie around 1e7 (32-bit numbers one apart): the distribution is that of their differences."""
    z, ids, t, w = _case(6, 5000, 8, "fp32", 24)
    near = z.round()
    for off in (1e7, -1.5e7):
        want = ops.topk_distill(near, ids, t, "jsd", return_log_probs=True)
        got = ops.topk_distill(near + off, ids, t, "jsd", return_log_probs=True)
        assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-6) for a, b in zip(got, want))
        grads = [torch.autograd.grad(ops.topk_distill(x, ids, t, "jsd"), x, w)[0] for x in (near.clone().requires_grad_(), (near + off).requires_grad_())]
        assert torch.allclose(*grads, rtol=2e-5, atol=1e-9)


@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd"])
def test_distill_renormalised_ids_far_behind(kl):
    """Ids whose mass is nothing to 64 bits beside the rest of the row still have their shares of one another's."""
    z, ids, t, w = _case(4, 700, 6, "fp32", 25)
    z.scatter_add_(1, ids, torch.full_like(t, -900.0))
    got = []
    for x, i, tt, ww in ((z, ids, t, w), (z.cpu().double(), ids.cpu(), t.cpu(), w.cpu())):      # (the CPU's log-softmax is in 64 bits)
        zl = x.detach().requires_grad_()
        loss = ops.topk_distill(zl, i, tt, kl, norm_mode="norm")
        got.append((loss.detach().cpu(), torch.autograd.grad(loss, zl, ww)[0].cpu().double()))
    # logits of 900 are off by 900 * 2^-24 in 32 bits, but the CPU reads the same ones: what is left are roundings of the results
    assert torch.allclose(got[0][0], got[1][0], rtol=1e-6, atol=1e-9)
    assert torch.allclose(got[0][1], got[1][1], rtol=1e-6, atol=1e-9)


@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd"])
def test_distill_shares_of_nothing(kl):
    z, ids, t, _ = _case(4, 50, 3, "fp32", 27)
    z[:2].scatter_(1, ids[:2], -math.inf)
    ids[1, 1:] = -1
    ids[2, 1:] = 70
    t[2] = -math.inf
    assert torch.isnan(ops.topk_distill(z, ids, t, kl, norm_mode="norm")).tolist() == [True, True, True, False]


def test_refusals_name_numbers():
    """The extension's own checks, for callers that come without the package's."""
    from relax_b200.ops import cuda as C

    m, ids = C._load(), torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    for bad, text in (((0, 1), "got 0"), ((2049, 1), "got 2049"), ((3, 0), "got 0"), ((3, 65537), "got 65537")):
        with pytest.raises(ValueError, match=text):
            m.expert_layout(ids, *bad)
    wide = torch.zeros(3, 1025, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="got 1025"):
        m.topk_distill(torch.zeros(3, 8, device="cuda"), wide, wide.float(), 0, 0, 0.5, -math.inf, 1.0, False)
    with pytest.raises(RuntimeError, match="code -1"):
        m.topk_distill(torch.zeros(3, 8, device="cuda"), ids, ids.float(), 9, 0, 0.5, -math.inf, 1.0, False)


@pytest.mark.parametrize("V", [(1 << 20) + 5, (1 << 23) - 1, 1 << 24])
def test_distill_vocabularies_of_any_size(V):
    """Parts of a row are as long as a bitmap in shared memory has room for."""
    z, ids, t, w = _case(1, 1000, 5, "bf16", 28)
    big = torch.full((1, V), -8.0, device="cuda", dtype=torch.bfloat16)
    big[:, -1000:] = z
    ids += V - 1000
    zl = big.requires_grad_()
    loss, lp = ops.topk_distill(zl, ids, t, "jsd", return_log_probs=True)
    (d,) = torch.autograd.grad(loss, zl, w)
    lse = torch.logaddexp(torch.logsumexp(z.double(), 1), torch.tensor(math.log(V - 1000.0) - 8.0, device="cuda", dtype=torch.float64))
    want = z.double().gather(1, ids - (V - 1000)) - lse[:, None]
    assert torch.allclose(lp.double(), want, rtol=1e-6, atol=2e-6)
    p, q = torch.cat([want.exp(), 1 - want.exp().sum(1, keepdim=True)], 1), torch.cat([t.double().exp(), 1 - t.double().exp().sum(1, keepdim=True)], 1)
    m = (p + q) / 2
    assert torch.allclose(loss.double(), ((p * (p / m).log() + q * (q / m).log()) / 2).sum(1), rtol=2e-5, atol=1e-7)
    slope = ((p / m).log() / 2)
    c = p[:, :5] * (slope[:, :5] - slope[:, 5:])
    assert torch.allclose(d[0, 0].double(), (-w[0] * c.sum() * math.exp(-8.0 - float(lse))).double(), rtol=1e-2)
    assert torch.equal(d[0, : V - 1000], d[0, 0].expand(V - 1000))
    with pytest.raises(ValueError, match="2.24"):
        ops.topk_distill(torch.empty(1, (1 << 24) + 1, device="cuda", dtype=torch.bfloat16), ids, t)


@pytest.mark.parametrize("R,V,K", [(1300, 515, 20), (1184, 1024, 256), (1184, 1024, 257), (1190, 4099, 8), (1200, 33, 33), (593, 4099, 512), (600, 2003, 513),
                                   (1184, 20001, 9), (700, 70007, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_distill_many_short_rows(R, V, K, dtype):
    """Blocks of fewer threads: rows of every alignment, up to the most ids that such blocks take and beyond."""
    z, ids, t, w = _case(R, V, K, dtype, 29)
    z[7, 1:] = -1e30
    z[8, :] = -1e9
    zl = z.detach().requires_grad_()
    loss, lp = ops.topk_distill(zl, ids, t, "jsd", return_log_probs=True)
    (d,) = torch.autograd.grad(loss, zl, w)
    some = torch.cat([torch.arange(20), torch.arange(R - 4, R)])
    zl = z[some.cuda()].clone().requires_grad_()      # the same rows, few of them: in blocks of more threads
    loss2, lp2 = ops.topk_distill(zl, ids[some.cuda()], t[some.cuda()], "jsd", return_log_probs=True)
    (d2,) = torch.autograd.grad(loss2, zl, w[some.cuda()])
    assert torch.allclose(loss[some.cuda()], loss2, rtol=1e-5, atol=1e-6) and torch.allclose(lp[some.cuda()], lp2, rtol=1e-6, atol=2e-6)
    assert torch.allclose(d[some.cuda()].float(), d2.float(), rtol=2 * _half_step(d.dtype) + 2e-5, atol=1e-8)
    plain = some[(some != 7) & (some != 8)].cuda()      # (which are those of the statement)
    _check(z[plain], ids[plain], t[plain], w[plain], kl="jsd")


def test_distill_rows_without_ids():
    """Nothing to compare: no loss and no gradient, whatever the row holds."""
    z, ids, t, w = _case(5, 1200, 6, "fp32", 26)
    ids[:4] = -1
    ids[3] = 1200
    z[0], z[1, 5], z[2] = -math.inf, math.nan, torch.finfo(torch.float32).min
    for norm in ("tail", "norm", "trunc"):
        for x, i, tt, ww in ((z, ids, t, w), (z.cpu(), ids.cpu(), t.cpu(), w.cpu())):
            zl = x.detach().requires_grad_()
            loss, lp = ops.topk_distill(zl, i, tt, "jsd", norm_mode=norm, return_log_probs=True)
            (d,) = torch.autograd.grad(loss, zl, ww)
            assert bool((loss[:4] == 0).all()) and bool((d[:4] == 0).all()) and bool((lp[:4] == -math.inf).all()) and float(loss[4]) > 0
    loss = ops.topk_distill(z, ids[:, :0], t[:, :0])
    assert bool((loss == 0).all())


@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd"])
def test_distill_a_single_renormalised_id(kl):
    """All mass is the one id's on both sides: exactly nothing to learn, wherever the other entries stand and however the id is clamped."""
    z, ids, t, w = _case(4, 900, 5, "fp32", 18)
    ids[:3, 1:] = -1
    ids[1] = ids[1].roll(2)
    t[1, 2] = -30.0
    for clamp in (None, -4.0):
        zl = z.detach().requires_grad_()
        loss = ops.topk_distill(zl, ids, t, kl, norm_mode="norm", log_prob_min_clamp=clamp)
        (d,) = torch.autograd.grad(loss, zl, w)
        assert bool((loss[:3] == 0).all()) and bool((d[:3] == 0).all()) and float(loss[3]) > 0


def test_distill_mixture_at_its_ends():
    z, ids, t, w = _case(20, 3001, 8, "bf16", 19)
    for alpha, kl in ((0.0, "reverse_kl"), (1.0, "forward_kl")):
        assert torch.equal(ops.topk_distill(z, ids, t, "jsd", alpha), ops.topk_distill(z, ids, t, kl))


def test_fused_head_of_frozen_weights():
    """A head that does not learn keeps its buffer, hidden states that need no gradient get none."""
    g = _gen(21)
    h = torch.randn(33, 64, device="cuda", generator=g).bfloat16()
    weight = torch.randn(512, 64, device="cuda", generator=g).bfloat16()
    _, ids, t, w = _case(33, 512, 6, "bf16", 22)
    want = []
    for freeze in (False, True):
        hl, wl = h.detach().requires_grad_(), weight.detach().requires_grad_(not freeze)
        wl.main_grad = torch.full((512, 64), 0.25, device="cuda")
        (ops.fused_lm_head_topk_distill(hl, wl, ids, t, chunk_size=16) * w).sum().backward()
        want.append(hl.grad)
        assert bool((wl.main_grad == 0.25).all()) == freeze
        learned = wl.main_grad if not freeze else learned
    assert torch.equal(*want)
    wl = weight.detach().requires_grad_()
    wl.main_grad = torch.full((512, 64), 0.25, device="cuda")
    (ops.fused_lm_head_topk_distill(h, wl, ids, t, chunk_size=16) * w).sum().backward()
    assert torch.equal(wl.main_grad, learned)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_distill_masks_of_the_lowest_value(dtype):
    """A mask may leave some tokens, or none: rows of nothing but the type's lowest value are uniform."""
    z, ids, t, w = _case(5, 1003, 7, dtype, 14)
    low = torch.finfo(DT[dtype]).min
    z[0] = low
    z[1, 10:] = low
    z[2, ::2] = low
    z[3, :] = -math.inf
    z[3, 5] = 1.0
    ids[1, :3] = torch.tensor([3, 500, 9], device="cuda")
    for norm, temperature in (("tail", 1.0), ("norm", 1.0), ("trunc", 0.5)):
        zl = z.detach().requires_grad_()
        loss = ops.topk_distill(zl, ids, t, "forward_kl" if norm == "trunc" else "jsd", norm_mode=norm, temperature=temperature)
        (d,) = torch.autograd.grad(loss, zl, w)
        r = [0, 1, 2, 4]
        zz = torch.where(z.double() <= -1e38, z.double() / 2 ** 20, z.double()) if dtype != "fp16" else z.double()      # (the same rows in exact arithmetic)
        want, d_want, _ = O.distill(zz[r], ids[r], t[r], w[r], "forward_kl" if norm == "trunc" else "jsd", 0.5, norm, temperature)
        fine = torch.isfinite(want)
        assert torch.allclose(loss[r].double().cpu()[fine], want[fine], rtol=1e-5, atol=1e-5)
        got = d[r].double().cpu()[fine]
        assert float((got - d_want[fine]).abs().max()) <= 2 * _half_step(DT[dtype]) * float(d_want[fine].abs().max()) + 1e-5
    lp = ops.topk_distill(z, ids, t, return_log_probs=True)[1]
    assert torch.allclose(lp[0], torch.full((7,), -math.log(1003.0), device="cuda"), atol=1e-5)


def test_distill_log_probs():
    z, ids, t, _ = _case(6, 5000, 20, "bf16", 3)
    ids[2, 4:] = -1
    _, lp = ops.topk_distill(z, ids, t, return_log_probs=True)
    want = torch.log_softmax(z.double(), 1).gather(1, ids.clamp_min(0))
    assert torch.equal(torch.isinf(lp), ids < 0)
    there = ids >= 0
    # the sum's error (2^-22 and A 2^-23 with |A| < 60, 45 additions) and the value's own rounding
    assert ((lp.double() - want).abs()[there] <= 2.0 ** -22 + 170 * F + F * want.abs()[there]).all()


def test_distill_captured():
    """Forward and backward in a graph, replayed on other inputs; the small kernel follows the streaming one as a programmatic dependent."""
    z, ids, t, w = _case(40, 20000, 16, "bf16", 9)
    zl = z.clone().requires_grad_()

    def both():
        loss, lp = ops.topk_distill(zl, ids, t, "jsd", return_log_probs=True)
        return loss, lp, torch.autograd.grad(loss, zl, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (1, 2, 3):
        other, ids2, t2, w2 = _case(40, 20000, 16, "bf16", 20 + seed)
        with torch.no_grad():
            zl.copy_(other)
        ids.copy_(ids2), t.copy_(t2), w.copy_(w2)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        assert all(torch.equal(a, b) for a, b in zip(got, both()))


def test_distill_gradient_against_differences():
    z, ids, t, w = _case(4, 777, 9, "fp32", 15)
    v = torch.randn(z.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    for kl in ("reverse_kl", "forward_kl", "jsd", "low_var_kl"):
        zz = z.clone().requires_grad_()
        (d,) = torch.autograd.grad(ops.topk_distill(zz, ids, t, kl), zz, w)
        h = 1e-5
        up, dn = (O.distill(z.double().cpu() + e * v, ids, t, w, kl)[0] for e in (h, -h))
        slope = float(((up - dn) / (2 * h) * w.cpu()).sum())
        dv = d.double().cpu() * v
        assert abs(float(dv.sum()) - slope) <= 1e-5 * float(dv.abs().sum() + 1.0), kl


def test_fused_head_distill():
    g = _gen(21)
    R, V, H, K = 300, 4096, 256, 16
    _, ids, t, w = _case(R, V, K, "fp32", 2)
    h = torch.randn(R, H, device="cuda", generator=g).bfloat16().requires_grad_()
    wt = (torch.randn(V, H, device="cuda", generator=g) * 0.1).bfloat16().requires_grad_()
    loss = ops.fused_lm_head_topk_distill(h, wt, ids, t, "jsd", chunk_size=128)
    d_h, d_w = torch.autograd.grad(loss, [h, wt], w)
    hd, wd = h.detach().double().requires_grad_(), wt.detach().double().requires_grad_()
    from relax_b200.ops import reference as ref

    ld = ref.topk_distill(hd @ wd.t(), ids, t, "jsd", 0.5, "tail", 1.0, None, False)
    assert torch.allclose(loss, ld, rtol=1e-4, atol=1e-5)
    e_h, e_w = torch.autograd.grad(ld, [hd, wd], w)
    for got, want in ((d_h, e_h), (d_w, e_w)):
        # d logits and the product are rounded to bf16 (2^-8 each) among terms of the product's size
        assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -7
    wt.main_grad = torch.zeros(V, H, device="cuda")
    h2 = h.detach().requires_grad_()
    ops.fused_lm_head_topk_distill(h2, wt, ids, t, "jsd", chunk_size=300).backward(w)
    assert wt.grad is None and float((wt.main_grad.double() - e_w).norm() / e_w.norm()) < 2.0 ** -7
    assert float((h2.grad.double() - e_h).norm() / e_h.norm()) < 2.0 ** -7


# --------------------------------------------------------------------------- far offsets, one gradient only


def test_offsets_beyond_32_bits():
    g = _gen(3)
    # a buffer of 2.2e9 elements
    T, k, E, H = 66000, 8, 16, 4096
    ids = torch.randint(0, E, (T, k), device="cuda", generator=g)
    rows = ops.expert_layout(ids, E)
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    srt = ops.expert_dispatch(x, rows)
    assert srt.numel() > 2 ** 31
    last = int(rows.dest[:, 0].argmax())
    assert torch.equal(srt[rows.dest[last].long()], x[last].expand(k, H)) and torch.equal(srt[int(rows.dest[0, 0])], x[0])
    w = torch.full((T, k), 0.125, device="cuda")
    out = ops.expert_combine(srt, w, rows)
    assert torch.equal(out[[0, last, T - 1]], x[[0, last, T - 1]])            # eight eighths of a row
    del srt, out
    # logits of 2.4e9 elements: the last rows are those of a small call
    R, V, K = 18000, 131072, 4
    z = torch.empty(R, V, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    ids = torch.randint(0, V, (R, K), device="cuda", generator=g)
    t = torch.full((R, K), -3.0, device="cuda")
    zl = z.requires_grad_()
    loss = ops.topk_distill(zl, ids, t)
    (d,) = torch.autograd.grad(loss.sum(), zl)
    small = z.detach()[-3:].clone().requires_grad_()
    part = ops.topk_distill(small, ids[-3:], t[-3:])
    (ds,) = torch.autograd.grad(part.sum(), small)
    assert torch.allclose(part, loss[-3:], rtol=1e-5, atol=1e-6) and torch.allclose(ds.float(), d[-3:].float(), rtol=2.0 ** -7, atol=1e-7)
    del z, zl, d, loss
    # a table of 2.2e9 elements
    table = torch.zeros(550000, 4096, device="cuda", dtype=torch.bfloat16)
    table[-1] = 1.0
    tok = torch.tensor([549999, 0, 549999, 123], device="cuda")
    leaf = table.requires_grad_()
    out = ops.embedding(tok, leaf)
    assert bool((out[0] == 1).all()) and not out[1].any()
    (d,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert bool((d[549999] == 2).all()) and bool((d[0] == 1).all()) and bool((d[123] == 1).all()) and int(d.count_nonzero()) == 3 * 4096


def test_gradients_are_given_once():
    z, ids, t, w = _case(3, 50, 4, "fp32", 1)
    zl = z.requires_grad_()
    wl = w.requires_grad_()
    (d,) = torch.autograd.grad(ops.topk_distill(zl, ids, t), zl, wl, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        d.sum().backward()
    rows = ops.expert_layout(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 2)
    x = torch.randn(4, 8, device="cuda").requires_grad_()
    up = torch.randn(rows.source.numel(), 8, device="cuda").requires_grad_()
    (d,) = torch.autograd.grad(ops.expert_dispatch(x, rows), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        d.sum().backward()


def test_combine_in_fp32_passes_gradients_on():
    g = _gen(4)
    ids = torch.randint(0, 5, (60, 3), device="cuda", generator=g)
    rows = ops.expert_layout(ids, 5)
    y = torch.randn(rows.source.numel(), 40, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.rand(60, 3, device="cuda", generator=g).bfloat16().requires_grad_()
    up = torch.randn(60, 40, device="cuda", generator=g).bfloat16()
    a = torch.autograd.grad(ops.expert_combine(y, w, rows, torch.float32), [y, w], up.float())
    b = torch.autograd.grad(ops.expert_combine(y, w, rows), [y, w], up)
    assert a[0].dtype == torch.bfloat16 and a[1].dtype == torch.bfloat16 and all(torch.equal(p, q) for p, q in zip(a, b))


def test_calls_of_two_threads():
    """Threads on streams of their own: no workspace, counter or limit is shared."""
    import threading

    g = _gen(6)
    cases = []
    for n, E in ((3000, 2048), (16000, 64)):
        ids = torch.randint(0, E, (n, 2), device="cuda", generator=g)
        x = torch.randn(n, 64, device="cuda", generator=g).bfloat16()
        tok = torch.randint(0, 700, (n,), device="cuda", generator=g)
        cases.append((ids, E, x, tok, torch.randn(n, 64, device="cuda", generator=g).bfloat16(), torch.randn(n // 50, 1000, device="cuda", generator=g)))

    def run(ids, E, x, tok, dy, z):
        rows = ops.expert_layout(ids, E)
        out = [rows.dest, ops.expert_combine(ops.expert_dispatch(x, rows), None, rows)]
        table = torch.zeros(700, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
        out += torch.autograd.grad(ops.embedding(tok, table), table, dy)
        at = tok[: 4 * z.shape[0]].view(-1, 4)
        return out + [ops.topk_distill(z, at, torch.full(at.shape, -4.0, device="cuda"))]

    want = [[t.clone() for t in run(*c)] for c in cases]
    torch.cuda.synchronize()
    got, failed = {}, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = run(*cases[i])
            s.synchronize()
        except Exception as e:   # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not failed, failed
    assert all(torch.equal(a, b) for i in range(2) for a, b in zip(want[i], got[i]))


# --------------------------------------------------------------------------- together


def test_step_of_a_routed_student():
    """Embedding, routed experts and the distillation loss of one step on the GPU in bf16 against the same layers in 64-bit plain torch."""
    g = _gen(33)
    T, V, H, E, k, Fh, K = 300, 2048, 256, 8, 2, 128, 12
    tok = torch.randint(0, V, (T,), device="cuda", generator=g)
    mk = lambda *s, m=1.0: (torch.randn(*s, device="cuda", generator=g) * m).bfloat16().requires_grad_()      # noqa: E731
    table, w1, w2, head = mk(V, H), mk(E, 2 * Fh, H, m=0.06), mk(E, H, Fh, m=0.1), mk(V, H, m=0.08)
    idx = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(T)])
    gate = torch.rand(T, k, device="cuda", generator=g).requires_grad_()
    _, ids, teacher, w = _case(T, V, K, "fp32", 3)

    from relax_b200.models.moe import experts_mlp

    x = ops.embedding(tok, table, 2.0)
    h = x + experts_mlp(x, idx, gate, w1, w2)
    loss = (ops.fused_lm_head_topk_distill(h, head, ids, teacher) * w).mean()
    grads = torch.autograd.grad(loss, [table, w1, w2, head, gate])

    D = [p.detach().double().requires_grad_() for p in (table, w1, w2, head, gate)]
    xd = D[0][tok] * 2.0
    gu = torch.einsum("th,tknh->tkn", xd, D[1][idx])
    act = torch.nn.functional.silu(gu[..., :Fh]) * gu[..., Fh:]
    hd = xd + (torch.einsum("tkf,tkhf->tkh", act, D[2][idx]) * D[4][..., None]).sum(1)
    z = hd @ D[3].t()
    lp = torch.log_softmax(z, 1).gather(1, ids)
    p, q = lp.exp(), teacher.double().exp()
    rp, rq = 1 - p.sum(1), 1 - q.sum(1)
    ld = (((p * (lp - teacher.double())).sum(1) + rp * (rp.log() - rq.log())) * w).mean()
    want = torch.autograd.grad(ld, D)
    assert abs(float(loss) - float(ld)) < 2e-2 * abs(float(ld))      # bf16 activations: four roundings of 2^-8 in front of the logits
    for got, ref in zip(grads, want):
        assert float((got.double() - ref).norm() / ref.norm()) < 5e-2, got.shape


@pytest.mark.parametrize("selection", ["teacher_topk", "student_topk", "union"])
def test_loss_mode_of_a_routed_student(tmp_path, monkeypatch, selection):
    """The training loop with ``--opd-loss-coef`` on top ids: every operator of this file in one step, as a user runs them."""
    import dataclasses

    from relax_b200.checkpoint import hf as H
    from relax_b200.config.arguments import parse_args
    from relax_b200.models import config as MC
    from relax_b200.models.transformer import GPTModel
    from relax_b200.orchestration.controller import Controller

    cfg = dataclasses.replace(MC.get_config("tiny-moe"), name="tiny-moe-wide-heads", head_dim=128, vocab_size=1024, dtype="bf16")
    monkeypatch.setitem(MC.PRESETS, cfg.name, cfg)
    teacher = GPTModel(cfg, seed=77)
    d = str(tmp_path / "teacher")
    H.save_hf_checkpoint(d, cfg, H.convert_state_to_hf(cfg, {k: v.detach() for k, v in teacher.named_parameters()}))
    a = parse_args(["--model-name", cfg.name, "--colocate", "--rollout-batch-size", "2", "--n-samples-per-prompt", "2", "--global-batch-size", "4",
                    "--num-rollout", "1", "--rollout-max-response-len", "24", "--use-opd", "--opd-teacher-load", d, "--lr", "1e-3", "--opd-loss-coef", "1.0",
                    "--opd-only-reward", "--opd-token-selection", selection, "--opd-log-prob-top-k", "16", "--opd-kl-type", "jsd"])
    c = Controller(a, device="cuda")
    actor, seen = c.runner.actor, {}
    plain = actor._distill_batch
    actor._distill_batch = lambda batch, ids: seen.setdefault("made", plain(batch, ids))
    hist = c.runner.step()
    made = seen["made"]
    assert made["divergence"].dtype == torch.float32 and bool((made["divergence"] >= 0).all())
    assert math.isfinite(hist["grad_norm"]) and hist["grad_norm"] > 0 and hist["opd_loss"] > 0
    assert hist["pg_loss"] == 0.0 and hist["loss"] == pytest.approx(hist["opd_loss"], rel=1e-6)
    assert made["ids"].shape[1] == 16 if selection != "union" else 16 < made["ids"].shape[1] <= 32
    assert c.runner.step()["opd_loss"] > 0
    c.runner.close()


@pytest.mark.parametrize("H,pitch", [(40, 40), (264, 264), (33, 33), (40, 44), (7, 9)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_combine_in_fp32_keeps_the_bits_of_its_gradient(dtype, H, pitch):
    """A sum kept in 32 bits takes a gradient in 32 bits: numbers that 16 bits round (and, in fp16, that they cannot hold)."""
    g, T, k, E = _gen(41), 90, 3, 5
    ids = torch.randint(-1, E, (T, k), device="cuda", generator=g)
    rows = ops.expert_layout(ids, E)
    cap = rows.source.numel()
    y = torch.randn(cap, H, device="cuda", generator=g).to(DT[dtype]).requires_grad_()
    w = (0.001 + 0.01 * torch.rand(T, k, device="cuda", generator=g)).requires_grad_()
    up = (1e5 * torch.randn(T, pitch, device="cuda", generator=g))[:, :H]
    d_y, d_w = torch.autograd.grad(ops.expert_combine(y, w, rows, torch.float32), [y, w], up)
    (plain,) = torch.autograd.grad(ops.expert_combine(y, None, rows, torch.float32), y, up / 1e5)
    half, dest = _half_step(DT[dtype]), rows.dest.cpu()
    u, yc, wc = up.double().cpu(), y.detach().double().cpu(), w.detach().double().cpu()
    want_y, want_p, want_w, size_w = (torch.zeros(*s, dtype=torch.float64) for s in ((cap, H), (cap, H), (T, k), (T, k)))
    for t in range(T):
        for j in range(k):
            d = int(dest[t, j])
            if d >= 0:
                want_y[d], want_p[d] = u[t] * wc[t, j], (up[t] / 1e5).double().cpu()
                want_w[t, j], size_w[t, j] = (u[t] * yc[d]).sum(), (u[t] * yc[d]).abs().sum()
    _within(d_y, want_y, (half + 2 * F) * want_y.abs() + 2.0 ** -25, "d y")             # a product in 32 bits, one rounding to 16
    _within(plain, want_p, half * want_p.abs() + 2.0 ** -25, "d y of a plain sum")
    _within(d_w, want_w, (H + 1) * F * size_w, "d weights")                             # (a rounding per term, in any order)


@pytest.mark.parametrize("H,k", [(264, 3), (33, 11)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_combine_gives_the_gradients_that_are_asked_for(dtype, H, k):
    """Rows are neither kept for weights that are fixed nor written for rows that are; what is given is what both together give."""
    g, T, E = _gen(42), 70, 5
    rows = ops.expert_layout(torch.randint(-1, E, (T, k), device="cuda", generator=g), E)
    y = torch.randn(rows.source.numel(), H, device="cuda", generator=g).to(DT[dtype])
    w, up = torch.rand(T, k, device="cuda", generator=g), torch.randn(T, H, device="cuda", generator=g).to(DT[dtype])
    yl, wl = y.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(ops.expert_combine(yl, wl, rows), [yl, wl], up)
    kept = yl * 1.0
    out = ops.expert_combine(kept, w, rows)
    with torch.no_grad():
        kept.zero_()                          # (an error in the backward pass, if it were kept for it)
    (d_y,) = torch.autograd.grad(out, yl, up)
    assert torch.equal(d_y, want[0])
    before = torch.cuda.memory_allocated()
    out = ops.expert_combine(y, wl, rows)
    torch.cuda.reset_peak_memory_stats()
    (d_w,) = torch.autograd.grad(out, wl, up)
    assert torch.equal(d_w, want[1])
    assert torch.cuda.max_memory_allocated() - before < y.numel() * y.element_size()
    (d_w,) = torch.autograd.grad(ops.expert_combine(yl, wl, rows), wl, up)      # only one of two is asked for
    assert torch.equal(d_w, want[1])


@pytest.fixture
def status():
    """The device's status word, clean before and after."""
    from relax_b200.ops import cuda as C

    C.check_error_flag()
    yield C.check_error_flag
    C.err_flag().zero_()


@pytest.mark.parametrize("cols,dtype", [(264, "bf16"), (520, "bf16"), (33, "fp32")])
@pytest.mark.parametrize("bad", [-1, 50, 1 << 40, -(1 << 40)])
def test_tokens_outside_a_whole_table_are_noted(status, cols, dtype, bad):
    g = _gen(43)
    table = torch.randn(50, cols, device="cuda", generator=g).to(DT[dtype]).requires_grad_()
    tok = torch.randint(0, 50, (700,), device="cuda", generator=g)
    want = ops.embedding(tok, table, whole=True)
    assert torch.equal(want, table[tok])
    status()
    tok[699] = bad
    out = ops.embedding(tok, table)                       # a shard's table: others have this token
    status()
    assert torch.equal(out[:699], want[:699]) and not out[699].any()
    out = ops.embedding(tok, table, whole=True)
    with pytest.raises(RuntimeError, match="status 4"):
        status()
    status()
    assert torch.equal(out[:699], want[:699]) and not out[699].any()


@pytest.mark.parametrize("T,k,E", [(5, 2, 4), (1, 8, 128), (30000, 3, 64)])
def test_expert_ids_outside_a_whole_table_are_noted(status, T, k, E):
    ids = torch.randint(0, E, (T, k), device="cuda", generator=_gen(44))
    rows = ops.expert_layout(ids, E, whole=True)
    status()
    assert torch.equal(rows.dest, ops.expert_layout(ids, E).dest)
    for bad in (-1, E):
        ids[T - 1, k - 1] = bad
        assert int(ops.expert_layout(ids, E).dest[T - 1, k - 1]) == -1
        status()
        ops.expert_layout(ids, E, whole=True)
        with pytest.raises(RuntimeError, match="status 4"):
            status()
        status()


def test_training_step_stops_at_a_token_outside_the_vocabulary(status):
    """Before its weights move, as indexing would have stopped it."""
    import dataclasses

    from relax_b200.algo.loss import LossConfig
    from relax_b200.models.config import get_config
    from relax_b200.train.actor import TrainActor, TrainConfig
    from relax_b200.train.optimizer import OptimizerConfig

    mcfg = dataclasses.replace(get_config("tiny-moe"), head_dim=128, vocab_size=1024, dtype="bf16")
    cfg = TrainConfig(advantage_estimator="grpo", global_batch_size=2, n_samples_per_prompt=2, loss=LossConfig(), optim=OptimizerConfig(lr=1e-3))
    actor = TrainActor(mcfg, cfg, role="actor", device="cuda")
    batch = lambda first: {"tokens": [[first, 5, 6, 7, 8, 9], [3, 5, 6, 7, 8, 10]], "response_lengths": [3, 3],      # noqa: E731
                           "loss_masks": [[1.0] * 3] * 2, "rewards": [1.0, 0.0]}
    before = actor.param_buf.clone()
    with pytest.raises(RuntimeError, match="status 4"):
        actor.train(0, batch(1024))
    assert torch.equal(actor.param_buf, before)
    assert math.isfinite(actor.train(1, batch(4))["grad_norm"]) and not torch.equal(actor.param_buf, before)


@pytest.mark.parametrize("V,K,whole", [(151936, 512, True), (151936, 513, False), (151936, 1024, False), (32003, 600, True)])
def test_distill_rows_of_many_ids_are_shared_out(V, K, whole):
    """700 rows are two waves of whole rows, the second mostly empty: small blocks take them in one, and where a row is long and has more ids
    than those hold, several blocks share it."""
    from relax_b200.ops import cuda as C

    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("waves of 148 multiprocessors")
    R = 700
    z = torch.randn(R, V, device="cuda", generator=_gen(45)).bfloat16()
    ids = torch.arange(K, device="cuda").expand(R, K).contiguous() * 7
    t = torch.full((R, K), -9.0, device="cuda")
    loss, kept = C._load().topk_distill_rows(z, ids, t, 0, 0, 0.5, -math.inf, 1.0)
    parts = (kept.numel() - R * K) // (4 * R) - 1      # (four statistics of a row, two 64-bit numbers of a part)
    assert (parts == 1) == whole
    few = ops.topk_distill(z[:3], ids[:3], t[:3])
    assert torch.allclose(loss[:3], few, rtol=1e-5, atol=1e-6)


def test_fused_head_holds_one_piece_of_logits():
    g = _gen(46)
    R, V, H, K, chunk = 1400, 32768, 64, 6, 512
    h, wt = torch.randn(R, H, device="cuda", generator=g).bfloat16().requires_grad_(), torch.randn(V, H, device="cuda", generator=g).bfloat16().requires_grad_()
    wt.main_grad = torch.zeros(V, H, device="cuda")
    ids, t = torch.arange(K, device="cuda").expand(R, K).contiguous(), torch.full((R, K), -3.0, device="cuda")
    for _ in range(2):      # (the second time without first calls' workspaces)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        loss = ops.fused_lm_head_topk_distill(h, wt, ids, t, chunk_size=chunk)
        forward = torch.cuda.max_memory_allocated() - before
        torch.cuda.reset_peak_memory_stats()
        loss.sum().backward()
        backward = torch.cuda.max_memory_allocated() - before
    piece = chunk * V
    small = 4 << 20      # (hidden states, their gradient, slopes of the ids)
    assert forward <= 4 * piece + small and backward <= (4 + 2) * piece + small


def test_model_takes_tokens_from_the_host():
    """As indexing a weight did."""
    import dataclasses

    from relax_b200.models.config import get_config
    from relax_b200.models.transformer import GPTModel

    m = GPTModel(dataclasses.replace(get_config("tiny"), dtype="bf16"), device="cuda", seed=1)
    tok = torch.tensor([3, 1023, 0, 3])
    emb = m.embedding.word_embeddings
    out = emb(tok, False)
    assert torch.equal(out, emb.weight[tok.cuda()])
    up = torch.randn(out.shape, device="cuda").bfloat16()
    assert torch.equal(*(torch.autograd.grad(emb(t, False), emb.weight, up)[0] for t in (tok, tok.cuda())))


def test_more_experts_than_a_block_counts(status):
    g = _gen(47)
    ids = torch.randint(0, 3000, (500, 2), device="cuda", generator=g)
    x, w = torch.randn(500, 64, device="cuda", generator=g).bfloat16(), torch.rand(500, 2, device="cuda", generator=g)
    rows = ops.expert_layout(ids.int(), 3000, 16, whole=True)
    status()
    dest, source, tiles, bounds = O.layout(ids.cpu(), 3000, 16)
    assert rows.dest.reshape(-1).tolist() == dest and rows.source.tolist() == source and rows.tile_expert.tolist() == tiles and rows.expert_rows.tolist() == bounds
    assert torch.equal(ops.expert_combine(ops.expert_dispatch(x, rows), None, rows, torch.float32), 2.0 * x.float())
    ids[7, 1] = 3000
    assert int(ops.expert_layout(ids, 3000).dest[7, 1]) == -1
    status()
    ops.expert_layout(ids, 3000, whole=True)
    with pytest.raises(RuntimeError, match="status 4"):
        status()


def test_serving_forms_in_inference_mode():
    g = _gen(48)
    ids, tok = torch.randint(0, 4, (64, 2), device="cuda", generator=g), torch.randint(0, 64, (40,), device="cuda", generator=g)
    x, w = torch.randn(64, 72, device="cuda", generator=g).bfloat16(), torch.rand(64, 2, device="cuda", generator=g)
    did, t = torch.randint(0, 72, (64, 3), device="cuda", generator=g), torch.full((64, 3), -2.0, device="cuda")
    leaf = x.clone().requires_grad_()

    def run():
        rows = ops.expert_layout(ids, 4)
        y = ops.expert_dispatch(leaf, rows)
        return [rows.dest, rows.source, y, ops.expert_combine(y, w, rows), ops.embedding(tok, leaf, 2.0, whole=True),
                *ops.topk_distill(leaf, did, t, return_log_probs=True)]

    want = [v.detach().clone() for v in run()]
    with torch.inference_mode():
        got = run()
    assert all(v.is_inference() for v in got) and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("T,k,E,load", [(1, 8, 16, "even"), (5, 2, 300, "even"), (300, 2, 4, "one"), (257, 3, 7, "steep"), (128, 1, 2, "one"), (700, 8, 64, "even")])
def test_expert_products_on_their_layout(T, k, E, load):
    """Both products and all gradients on the buffer that the models use: no room to spare, tiles without rows, experts without rows."""
    from relax_b200.models.moe import experts_mlp

    g, H, Fh = _gen(49), 128, 64
    if load == "one":
        idx = torch.full((T, k), E - 1, device="cuda")
    elif load == "steep":
        idx = (torch.rand(T, k, device="cuda", generator=g) ** 4 * E).long()
    else:
        idx = torch.rand(T, E, device="cuda", generator=g).topk(k, -1).indices
    mk = lambda *s, m=1.0: (torch.randn(*s, device="cuda", generator=g) * m).bfloat16().requires_grad_()      # noqa: E731
    x, w1, w2, gate = mk(T, H), mk(E, 2 * Fh, H, m=0.09), mk(E, H, Fh, m=0.12), torch.rand(T, k, device="cuda", generator=g).requires_grad_()
    out = experts_mlp(x, idx, gate, w1, w2, whole=True)
    up = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    got = [out, *torch.autograd.grad(out, [x, gate, w1, w2], up)]
    D = [p.detach().double().requires_grad_() for p in (x, gate, w1, w2)]
    gu = torch.einsum("th,tknh->tkn", D[0], D[2][idx])
    y = torch.einsum("tkf,tkhf->tkh", torch.nn.functional.silu(gu[..., :Fh]) * gu[..., Fh:], D[3][idx])
    ref = (y * D[1][..., None]).sum(1)
    want = [ref, *torch.autograd.grad(ref, D, up.double())]
    for a, b in zip(got, want):      # five roundings to 16 bits in a row, 2^-8 each
        assert float((a.double() - b).norm()) <= 5 * 2.0 ** -8 * float(b.norm())
