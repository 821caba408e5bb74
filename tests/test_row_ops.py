"""Rows sorted by expert and back, the embedding with its gradient and the distillation divergence on the CPU: statements against one-row-at-a-time
oracles, refusals, and the paths of the framework that call them."""
import math

import pytest
import torch

import oracle_rows as O
from relax_b200 import ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("align", [1, 4, 128])
@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 3, 5), (40, 3, 7), (33, 2, 300)])
def test_expert_rows_statement(T, k, E, align):
    g = _gen(T + E)
    ids = torch.randint(-2, E + 2, (T, k), generator=g)
    rows = ops.expert_layout(ids, E, align)
    dest, source, tiles, bounds = O.layout(ids, E, align)
    assert rows.dest.reshape(-1).tolist() == dest and rows.source.tolist() == source and rows.expert_rows.tolist() == bounds
    assert (rows.tile_expert is None) == (align == 1)
    if align > 1:
        assert rows.tile_expert.tolist() == tiles
    x = torch.randn(T, 6, generator=g, dtype=torch.float32).requires_grad_()
    y = torch.randn(len(source), 6, generator=g).requires_grad_()
    w = torch.rand(T, k, generator=g).requires_grad_()
    srt, out = ops.expert_dispatch(x, rows), ops.expert_combine(y, w, rows)
    assert torch.equal(srt.double(), O.dispatch(x.detach(), source, k))
    want, size = O.combine(y.detach(), w.detach(), dest, k)
    assert ((out.double() - want).abs() <= (k + 1) * 2.0 ** -24 * size).all()
    d_s, d_o = torch.randn(srt.shape, generator=g), torch.randn(T, 6, generator=g)
    d_x, d_y, d_w = torch.autograd.grad([srt, out], [x, y, w], [d_s, d_o])
    want, size = O.combine(d_s, None, dest, k)
    assert ((d_x.double() - want).abs() <= (k + 1) * 2.0 ** -24 * size).all()
    for i, d in enumerate(dest):
        if d < 0:
            assert float(d_w.reshape(-1)[i]) == 0.0
        else:
            terms = d_o[i // k].double() * y[d].detach().double()
            assert abs(float(d_w.reshape(-1)[i]) - float(terms.sum())) <= 8 * 2.0 ** -24 * float(terms.abs().sum())
            assert torch.allclose(d_y[d], d_o[i // k] * w.detach().reshape(-1)[i], rtol=2.0 ** -23, atol=0)
    assert all((d_y[r] == 0).all() for r, s in enumerate(source) if s < 0)


def test_expert_rows_refusals():
    with pytest.raises(ValueError, match="int64 or int32"):
        ops.expert_layout(torch.zeros(3, 2), 4)
    with pytest.raises(ValueError, match="2048 experts"):
        ops.expert_layout(torch.zeros(3, 2, dtype=torch.int64), 0)
    with pytest.raises(ValueError, match="align"):
        ops.expert_layout(torch.zeros(3, 2, dtype=torch.int64), 4, 0)
    with pytest.raises(ValueError, match="at least one expert"):
        ops.expert_layout(torch.zeros(3, 0, dtype=torch.int64), 4)
    rows = ops.expert_layout(torch.zeros(3, 2, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="expert_dispatch"):
        ops.expert_dispatch(torch.zeros(4, 8), rows)
    with pytest.raises(ValueError, match="expert_combine"):
        ops.expert_combine(torch.zeros(5, 8), torch.ones(3, 2), rows)
    with pytest.raises(ValueError, match="weights"):
        ops.expert_combine(torch.zeros(rows.source.numel(), 8), torch.ones(2, 3), rows)


@pytest.mark.parametrize("scale", [1.0, 45.0])
@pytest.mark.parametrize("start", [0, 10])
def test_embedding_statement(scale, start):
    g = _gen(7)
    w = torch.randn(20, 5, generator=g).requires_grad_()
    tok = torch.randint(0, 40, (3, 11), generator=g)
    out = ops.embedding(tok, w, scale, start)
    dy = torch.randn(out.shape, generator=g)
    for i, t in enumerate(tok.reshape(-1).tolist()):
        here = 0 <= t - start < 20
        assert torch.equal(out.reshape(-1, 5)[i], w.detach()[t - start] * scale if here else torch.zeros(5))
    want, size = O.embedding_grad(tok, dy.reshape(-1, 5), 20, start, scale)
    (got,) = torch.autograd.grad(out, w, dy)
    assert ((got.double() - want).abs() <= 36 * 2.0 ** -24 * size).all()
    # into the optimizer's buffer
    w.main_grad = torch.full((20, 5), 0.5)
    ops.embedding(tok, w, scale, start).backward(dy)
    assert w.grad is None and torch.allclose(w.main_grad, got + 0.5, rtol=2.0 ** -20, atol=2.0 ** -20 * float(size.max()))
    with pytest.raises(ValueError, match="tokens"):
        ops.embedding(tok.float(), w)
    with pytest.raises(IndexError, match="table of 20 rows"):
        ops.embedding(tok, w, scale, start, whole=True)
    assert ops.embedding(tok[:0], w, whole=True).shape == (0, 11, 5)


def test_model_embedding_takes_the_configured_scale():
    import dataclasses

    from relax_b200.models.config import get_config
    from relax_b200.models.transformer import GPTModel

    cfg = dataclasses.replace(get_config("tiny"), embed_scale=3.0)
    m, plain = GPTModel(cfg, seed=1), GPTModel(get_config("tiny"), seed=1)
    tok = torch.tensor([1, 5, 1023])
    assert torch.equal(m.embedding.word_embeddings(tok, False), 3.0 * plain.embedding.word_embeddings(tok, False))


def _rows(R, V, K, seed, absent=True):
    g = _gen(seed)
    z = 3.0 * torch.randn(R, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)]) if R else torch.zeros(0, K, dtype=torch.int64)
    t = torch.log_softmax(2.0 * torch.randn(R, K + 1, generator=g), 1)[:, :K].contiguous()
    if absent and K > 1 and R > 1:
        ids[0, K // 2:] = -1
        ids[R - 1] = -1
    return z, ids, t, 0.5 + torch.rand(R, generator=g)


@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd", "low_var_kl"])
@pytest.mark.parametrize("norm", ["tail", "norm", "trunc"])
@pytest.mark.parametrize("clamp,temperature", [(None, 1.0), (-4.0, 0.7)])
def test_distill_statement(kl, norm, clamp, temperature):
    from relax_b200.algo import opd

    z, ids, t, w = _rows(5, 23, 6, 3)
    want, d_want, size = O.distill(z, ids, t, w, kl, 0.3, norm, temperature, clamp)
    z.requires_grad_()
    loss, lp = ops.topk_distill(z, ids, t, kl, 0.3, norm, temperature, clamp, return_log_probs=True)
    assert not lp.requires_grad
    # 64-bit arithmetic, one rounding to 32 bits
    assert ((loss.detach().double() - want).abs() <= 2.0 ** -24 * want.abs() + 1e-13 * size).all()
    (d,) = torch.autograd.grad(loss, z, w)
    assert ((d.double() - d_want).abs() <= 2.0 ** -23 * d_want.abs() + 1e-7 * size[:, None] * w[:, None]).all()
    away = ids < 0
    ref = (z.detach() / temperature).log_softmax(-1).gather(1, ids.clamp_min(0))
    assert torch.equal(torch.isinf(lp), away) and torch.allclose(lp[~away], ref[~away], atol=1e-5)
    # the same divergence as on gathered log-probs (32-bit arithmetic there, whose bin of all other mass loses digits)
    old = opd.token_kl(ref.masked_fill(away, 0.0), t, kl, 0.3, norm, clamp, mask=~away)
    assert torch.allclose(loss.detach(), old, atol=1e-4, rtol=1e-4)


def test_distill_gradient_against_differences():
    z, ids, t, w = _rows(4, 31, 5, 11)
    for kl in ("reverse_kl", "forward_kl", "jsd", "low_var_kl"):
        for norm in ("tail", "norm", "trunc"):
            zz = z.clone().requires_grad_()
            (d,) = torch.autograd.grad(ops.topk_distill(zz, ids, t, kl, 0.3, norm), zz, w)
            v = torch.randn(z.shape, generator=_gen(5), dtype=torch.float64)
            h = 1e-5
            up, dn = (O.distill(z.double() + e * v, ids, t, w, kl, 0.3, norm)[0] for e in (h, -h))
            slope = float(((up - dn) / (2 * h) * w).sum())
            # central differences: h^2 / 6 times the third derivative, of the order of the slope's terms
            assert abs(float((d.double() * v).sum()) - slope) <= 1e-5 * float((d.double() * v).abs().sum() + 1.0), (kl, norm)


def test_distill_edges_and_refusals():
    z, ids, t, _ = _rows(3, 9, 4, 1, absent=False)
    ids[1, 3] = ids[1, 0]                        # an id twice counts twice, as written
    want, _, _ = O.distill(z, ids, t, torch.ones(3), "reverse_kl", norm="trunc")
    assert torch.allclose(ops.topk_distill(z, ids, t, norm_mode="trunc").double(), want, rtol=1e-6)
    assert torch.equal(ops.topk_distill(z, torch.full_like(ids, 9), t), torch.zeros(3))
    assert ops.topk_distill(z, ids[:, :0], t[:, :0]).tolist() == [0.0] * 3
    t2 = t.clone()
    t2[0, 0] = -math.inf                         # the teacher rules a token out that the student gives mass
    assert torch.isinf(ops.topk_distill(z, ids, t2)[0]) and torch.isfinite(ops.topk_distill(z, ids, t2, "forward_kl")).all()
    for bad, match in ((dict(kl_type="kl"), "unknown divergence"), (dict(norm_mode="none"), "norm_mode"), (dict(alpha=1.5), "alpha"),
                       (dict(temperature=0.0), "temperature")):
        with pytest.raises(ValueError, match=match):
            ops.topk_distill(z, ids, t, **bad)
    with pytest.raises(ValueError, match="ids"):
        ops.topk_distill(z, ids[:2], t)
    with pytest.raises(ValueError, match="1024"):
        ops.topk_distill(z, torch.zeros(3, 1025, dtype=torch.int64), torch.zeros(3, 1025))
    with pytest.raises(ValueError, match="logits"):
        ops.topk_distill(z[0], ids, t)


def test_fused_head_distill_chunks():
    g = _gen(2)
    _, ids, t, w = _rows(7, 24, 4, 9)
    h, wt = torch.randn(7, 8, generator=g), torch.randn(24, 8, generator=g)
    outs = []
    for chunk in (3, 100):
        a, b = h.clone().requires_grad_(), wt.clone().requires_grad_()
        loss = ops.fused_lm_head_topk_distill(a, b, ids, t, "jsd", chunk_size=chunk)
        outs.append((loss.detach(), *torch.autograd.grad(loss, [a, b], w)))
    for x, y in zip(*outs):
        assert torch.allclose(x, y, atol=1e-5, rtol=1e-5)
    assert torch.allclose(outs[0][0], ops.topk_distill(h @ wt.t(), ids, t, "jsd"), atol=1e-6)
    assert ops.fused_lm_head_topk_distill(h[:0], wt, ids[:0], t[:0]).shape == (0,)


@pytest.mark.parametrize("selection", ["teacher_topk", "student_topk", "union"])
def test_loss_mode_on_top_ids(tmp_path, selection):
    """``--opd-loss-coef`` with a top-K selection: the step runs, the term is the only one that trains, and its gradient is that of the
    divergence of the policy's own logits."""
    from relax_b200.algo import opd
    from relax_b200.checkpoint import hf as H
    from relax_b200.config.arguments import parse_args
    from relax_b200.models.config import get_config
    from relax_b200.models.transformer import GPTModel
    from relax_b200.orchestration.controller import Controller

    cfg = get_config("tiny")
    teacher = GPTModel(cfg, seed=77)
    d = str(tmp_path / "teacher")
    H.save_hf_checkpoint(d, cfg, H.convert_state_to_hf(cfg, {k: v.detach() for k, v in teacher.named_parameters()}))
    a = parse_args(["--model-name", "tiny", "--colocate", "--rollout-batch-size", "2", "--n-samples-per-prompt", "2", "--global-batch-size", "4",
                    "--num-rollout", "1", "--rollout-max-response-len", "6", "--use-opd", "--opd-teacher-load", d, "--lr", "1e-3", "--opd-loss-coef", "1.0",
                    "--opd-only-reward", "--opd-token-selection", selection, "--opd-log-prob-top-k", "5", "--opd-kl-type", "jsd"])
    assert a.opd_kl_coef == 0.0
    c = Controller(a, device="cpu")
    actor = c.runner.actor
    seen = {}
    plain = actor._distill_batch
    actor._distill_batch = lambda batch, ids: seen.setdefault("made", plain(batch, ids))
    hist = c.runner.step()
    assert "opd_loss" in hist and math.isfinite(hist["grad_norm"]) and hist["grad_norm"] > 0
    assert hist["pg_loss"] == 0.0 and hist["loss"] == pytest.approx(hist["opd_loss"], abs=1e-6)
    made = seen["made"]
    assert made["divergence"].requires_grad and (made["divergence"] >= -1e-6).all() and made["ids"].shape == made["teacher"].shape
    assert selection == "union" or (made["ids"].shape[1] == 5 and (made["ids"] >= 0).all())
    c.runner.close()
    # the model's call against whole logits and the divergence on gathered log-probs
    m = GPTModel(cfg, seed=5)
    h = torch.randn(made["ids"].shape[0], cfg.hidden_size, generator=_gen(1))
    got = m.topk_distill(h, made["ids"], made["teacher"], 0.8, kl_type="jsd", alpha=0.5, norm_mode="tail")
    lp = torch.log_softmax(m.logits(h)[:, : cfg.vocab_size] / 0.8, -1).gather(1, made["ids"].clamp_min(0))
    want = opd.token_kl(lp, made["teacher"].masked_fill(made["ids"] < 0, 0.0), "jsd", 0.5, "tail", mask=made["ids"] >= 0)
    assert torch.allclose(got, want, atol=1e-5, rtol=1e-4)


@pytest.mark.parametrize("extra,match", [(["--tensor-model-parallel-size", "2"], "tp = cp = pp = 1"), (["--context-parallel-size", "2"], "tp = cp = pp = 1"),
                                         (["--opd-log-prob-top-k", "600"], "up to 512")])
def test_loss_mode_refusals(extra, match):
    from relax_b200.config.arguments import parse_args

    base = ["--model-name", "tiny", "--colocate", "--rollout-batch-size", "2", "--use-opd", "--opd-teacher-load", "somewhere", "--opd-loss-coef", "1.0",
            "--opd-token-selection", "union", "--opd-log-prob-top-k", "512"]
    assert parse_args(base).opd_loss_coef == 1.0
    with pytest.raises(ValueError, match=match):
        parse_args(base + extra)


def test_distill_temperatures():
    z, ids, t = _rows(3, 50, 4, 2)[:3]
    for bad in (0.0, -1.0, math.inf, math.nan, 1e-21):
        with pytest.raises(ValueError, match="temperature"):
            ops.topk_distill(z, ids, t, temperature=bad)


@pytest.mark.parametrize("norm", ["tail", "norm", "trunc"])
@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd", "low_var_kl"])
def test_distill_keeps_nan(kl, norm):
    """A row without a distribution (all masked, or a NaN among its logits) has no divergence."""
    z, ids, t, _ = _rows(4, 50, 4, 2, absent=False)
    z[1] = -math.inf
    z[2, 7] = math.nan
    loss = ops.topk_distill(z, ids, t, kl, norm_mode=norm)
    assert torch.isnan(loss).tolist() == [False, True, True, False]


@pytest.mark.parametrize("kl", ["reverse_kl", "forward_kl", "jsd"])
def test_distill_shares_of_nothing(kl):
    """Renormalising ids without any mass gives no shares, whether absent ids stand beside them or not."""
    z, ids, t, _ = _rows(4, 50, 3, 2, absent=False)
    z[:2].scatter_(1, ids[:2], -math.inf)
    ids[1, 1:] = -1
    ids[2, 1:] = 70
    t[2] = -math.inf
    loss = ops.topk_distill(z, ids, t, kl, norm_mode="norm")
    assert torch.isnan(loss).tolist() == [True, True, True, False]
    z = torch.full((1, 9), torch.finfo(torch.float32).min)       # ids far below absent ones share their mass all the same
    z[0, 8] = 0.0
    ids = torch.tensor([[3, -1, 5]])
    t = torch.tensor([[0.25, 0.5, 0.75]]).log()
    want = {"reverse_kl": 0.5 * math.log(0.5 / 0.25) + 0.5 * math.log(0.5 / 0.75), "forward_kl": 0.25 * math.log(0.5) + 0.75 * math.log(1.5)}
    if kl in want:
        assert float(ops.topk_distill(z, ids, t, kl, norm_mode="norm")) == pytest.approx(want[kl], rel=1e-6)


def test_extension_uses_the_process_s_cxx_runtime():
    """Two C++ runtimes in one process: a refusal that names a number would end it."""
    import os
    import shutil
    import subprocess

    from relax_b200.ops.build import SO_PATH

    if not (shutil.which("readelf") and os.path.exists(SO_PATH)):
        pytest.skip("readelf and a built extension")
    found = subprocess.run(["readelf", "-d", SO_PATH], capture_output=True, text=True, check=True).stdout
    assert "[libstdc++.so" in found


def test_rows_of_64_bits_keep_them():
    """A model in double precision on the CPU: sums, factors and gradients are in 64 bits, off by their own roundings only."""
    g, D = _gen(5), 2.0 ** -53
    ids = torch.randint(-1, 4, (30, 3), generator=g)
    rows = ops.expert_layout(ids, 4, 8)
    dest = rows.dest.reshape(-1).tolist()
    y = torch.randn(rows.source.numel(), 6, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.rand(30, 3, generator=g, dtype=torch.float64).requires_grad_()
    out = ops.expert_combine(y, w, rows)
    want, size = O.combine(y.detach(), w.detach(), dest, 3)
    assert out.dtype == torch.float64 and ((out - want).abs() <= 4 * D * size).all()
    assert torch.equal(ops.expert_combine(y, w, rows, torch.float32), out.float())
    up = torch.randn(30, 6, generator=g, dtype=torch.float64)
    d_y, d_w = torch.autograd.grad(out, [y, w], up)
    for i, d in enumerate(dest):
        if d >= 0:
            assert torch.equal(d_y[d], up[i // 3] * w.detach().reshape(-1)[i])
            terms = up[i // 3] * y[d].detach()
            assert abs(float(d_w.reshape(-1)[i] - terms.sum())) <= 12 * D * float(terms.abs().sum())
    table = torch.randn(9, 5, generator=g, dtype=torch.float64).requires_grad_()
    tok = torch.randint(-1, 10, (200,), generator=g)
    got = ops.embedding(tok, table, 1.0 / 3.0)
    here = (tok >= 0) & (tok < 9)
    assert torch.equal(got[here], table.detach()[tok[here]] * (1.0 / 3.0)) and not got[~here].any()
    dy = torch.randn(200, 5, generator=g, dtype=torch.float64)
    (d,) = torch.autograd.grad(got, table, dy)
    want, size = O.embedding_grad(tok, dy, 9, 0, 1.0 / 3.0)
    assert d.dtype == torch.float64 and ((d - want).abs() <= 210 * D * size).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_of_copied_rows_is_summed_in_32_bits(dtype):
    g, k = _gen(6), 8
    rows = ops.expert_layout(torch.randint(-1, 6, (20, k), generator=g), 6, 4)
    x = torch.randn(20, 5, generator=g).to(dtype).requires_grad_()
    up = torch.randn(rows.source.numel(), 5, generator=g).to(dtype)
    (d,) = torch.autograd.grad(ops.expert_dispatch(x, rows), x, up)
    want, size = O.combine(up, None, rows.dest.reshape(-1).tolist(), k)
    half = torch.finfo(dtype).eps / 2
    assert d.dtype == dtype and ((d.double() - want).abs() <= half * want.abs() + (1 + half) * (k + 1) * 2.0 ** -24 * size + 2.0 ** -25).all()


def test_fused_head_of_16_bit_weights_has_32_bit_logits():
    g = _gen(8)
    _, ids, t, w = _rows(7, 40, 4, 9)
    h, wt = (3 * torch.randn(7, 64, generator=g)).bfloat16().requires_grad_(), torch.randn(40, 64, generator=g).bfloat16().requires_grad_()
    loss = ops.fused_lm_head_topk_distill(h, wt, ids, t, chunk_size=3)
    hd, wd = h.detach().double().requires_grad_(), wt.detach().double().requires_grad_()
    want, _, size = O.distill(hd.detach() @ wd.detach().t(), ids, t, w)
    # a logit is off by its 64 products' roundings, the divergence by as much times its terms
    logit = 65 * 2.0 ** -24 * (hd.detach().abs() @ wd.detach().abs().t()).amax(1)
    assert loss.dtype == torch.float32 and ((loss.detach().double() - want).abs() <= 2.0 ** -24 * want.abs() + 4 * logit * size).all()
    d_h, d_w = torch.autograd.grad(loss, [h, wt], w)
    exact = ops.topk_distill(hd @ wd.t(), ids, t)
    e_h, e_w = torch.autograd.grad(exact, [hd, wd], w)
    assert d_h.dtype == d_w.dtype == torch.bfloat16
    for got, e in ((d_h, e_h), (d_w, e_w)):      # rounded to bf16 once, of a whole row's or (the head's, in pieces) three pieces' sums
        assert float((got.double() - e).norm() / e.norm()) < 3 * 2.0 ** -8


def test_teacher_gets_no_gradient():
    z, ids, t, w = _rows(4, 30, 5, 3)
    t.requires_grad_()
    assert not ops.topk_distill(z, ids, t, "jsd").requires_grad
    zl = z.clone().requires_grad_()
    d_z, d_t = torch.autograd.grad(ops.topk_distill(zl, ids, t, "jsd"), [zl, t], w, allow_unused=True)
    assert d_t is None and bool(d_z.any())


def test_whole_tables_of_experts_refuse_ids_outside():
    from relax_b200.models.moe import experts_mlp, grouped_swiglu_mlp

    g = _gen(9)
    ids = torch.tensor([[0, 3], [2, 1]])
    assert torch.equal(ops.expert_layout(ids, 4, 8, whole=True).dest, ops.expert_layout(ids, 4, 8).dest)
    assert ops.expert_layout(ids[:0], 4, whole=True).dest.shape == (0, 2)
    for bad in (-1, 4):
        ids[1, 1] = bad
        with pytest.raises(IndexError, match="of 4 experts"):
            ops.expert_layout(ids, 4, whole=True)
        assert int(ops.expert_layout(ids, 4).dest[1, 1]) == -1
    x, w1, w2 = torch.randn(2, 6, generator=g), torch.randn(4, 10, 6, generator=g), torch.randn(4, 6, 5, generator=g)
    with pytest.raises(IndexError, match="of 4 experts"):
        grouped_swiglu_mlp(x, torch.tensor([0, 4]), w1, w2)
    out = grouped_swiglu_mlp(x, torch.tensor([0, 4]), w1, w2, skip_foreign=True)
    assert not out[1].any() and torch.equal(out[:1], grouped_swiglu_mlp(x[:1], torch.tensor([0]), w1, w2))
    with pytest.raises(IndexError, match="of 4 experts"):
        experts_mlp(x, ids, torch.ones(2, 2), w1, w2, whole=True)
    assert experts_mlp(x[:0], ids[:0], torch.ones(0, 2), w1, w2, whole=True).shape == (0, 6)


def test_engine_refuses_prompts_outside_the_vocabulary():
    """The request alone: before it reaches the device, and without an end to the server or to what others run."""
    from relax_b200.models.config import get_config
    from relax_b200.rollout.engine import RolloutEngine, SamplingParams
    from relax_b200.rollout.http_server import EngineServer

    cfg = get_config("tiny")
    eng = RolloutEngine(cfg, device="cpu", dtype=torch.float32, num_kv_blocks=64, block_size=8, seed=3)
    for bad in ([3, cfg.vocab_size], [-1], [1 << 40, 2]):
        with pytest.raises(ValueError, match="outside the vocabulary of"):
            eng.add_request(bad, SamplingParams(max_new_tokens=2))
    with pytest.raises(ValueError, match="outside the vocabulary of"):
        eng.add_request([3], SamplingParams(max_new_tokens=2), resume_output=[cfg.vocab_size])
    assert not eng.has_work
    srv = EngineServer(eng)
    try:
        got = srv.generate({"input_ids": [[3, 5], [3, cfg.vocab_size], [0, cfg.vocab_size - 1]], "sampling_params": {"max_new_tokens": 3, "ignore_eos": True}})
        assert [len(d["output_ids"]) for d in got] == [3, 0, 3]
        assert "outside the vocabulary" in str(got[1]["finish_reason"])
    finally:
        srv.close()


def test_more_experts_than_a_block_counts():
    ids = torch.randint(-1, 5001, (300, 2), generator=_gen(10))
    rows = ops.expert_layout(ids, 5000, 8)
    dest, source, tiles, bounds = O.layout(ids, 5000, 8)
    assert rows.dest.reshape(-1).tolist() == dest and rows.source.tolist() == source and rows.tile_expert.tolist() == tiles and rows.expert_rows.tolist() == bounds
