"""Distillation on top ids as a loss term: whose experts route the teacher's passes, which rows reach the loss, and what the step trains on."""
import math

import pytest
import torch

from relax_b200.algo.loss import LossConfig
from relax_b200.models.config import get_config
from relax_b200.models.moe import RoutingReplay
from relax_b200.models.transformer import GPTModel
from relax_b200.train.actor import TrainActor, TrainConfig
from relax_b200.train.optimizer import OptimizerConfig

SEL = ["teacher_topk", "student_topk", "union"]


@pytest.fixture(autouse=True)
def _no_replay_left():
    yield
    RoutingReplay.end()
    RoutingReplay.per_sample = {}


def _actor(model="tiny-moe", micro=2, selection="teacher_topk", coef=1.0, lr=0.0, **kw):
    cfg = TrainConfig(advantage_estimator="grpo", global_batch_size=4, n_samples_per_prompt=2, use_dynamic_batch_size=False, micro_batch_size=micro,
                      pad_multiple=1, opd_token_selection=selection, opd_log_prob_top_k=5, opd_kl_type="jsd",
                      loss=LossConfig(opd_loss_coef=coef, opd_kl_type="jsd"), optim=OptimizerConfig(lr=lr), **kw)
    actor = TrainActor(get_config(model), cfg, role="actor", seed=0)
    g = torch.Generator().manual_seed(3)
    teacher = actor.param_buf + 0.1 * torch.randn(actor.param_buf.shape, generator=g)      # (the norms' weights too)
    actor.snapshots["teacher"] = teacher
    return actor


def _batch(actor, routed=False):
    g = torch.Generator().manual_seed(1)
    lens, rl = (12, 9, 14, 10), [5, 4, 6, 3]
    toks = [torch.randint(3, 1000, (n,), generator=g).tolist() for n in lens]
    batch = {"tokens": toks, "response_lengths": rl, "loss_masks": [[1.0] * r for r in rl], "rewards": [1.0, 0.0, 0.0, 1.0]}
    if routed:      # as recorded by an engine, other than what either router would choose
        c = actor.mcfg
        moe = [i for i in range(c.num_layers) if c.is_moe_layer(i)]
        batch["rollout_routed_experts"] = [torch.stack([torch.randperm(c.num_experts, generator=g)[: c.moe_top_k] for _ in range((n - 1) * len(moe))])
                                           .view(n - 1, len(moe), c.moe_top_k).tolist() for n in lens]
    return batch


def _teacher_alone(actor, batch, ids=None, k=5):
    """The teacher's top ids and log-probs, or its log-probs of given ids, by whole logits of one sample after the other, without replay."""
    m = GPTModel(actor.mcfg, seed=0)
    named = dict(actor.model.named_parameters())
    off = {id(p): o for p, o in actor._bound_params()}
    m.load_state_dict({n: actor.snapshots["teacher"][off[id(p)]: off[id(p)] + p.numel()].view_as(p) for n, p in named.items()}, strict=False)
    out = []
    for i, (t, r) in enumerate(zip(batch["tokens"], batch["response_lengths"])):
        with torch.no_grad():
            h = m(torch.tensor(t), torch.arange(len(t)), torch.tensor([0, len(t)], dtype=torch.int32), max_seqlen=len(t))
            lp = torch.log_softmax(m.logits(h)[len(t) - r - 1:len(t) - 1, : actor.mcfg.vocab_size].double(), -1)
        if ids is None:
            out.append(lp.topk(k, -1)[::-1])
        else:
            q = torch.as_tensor(ids[i])
            out.append((q, lp.gather(-1, q.clamp_min(0)).masked_fill(q < 0, -math.inf)))
    return out


@pytest.mark.parametrize("flags", [dict(use_routing_replay=True), dict(use_rollout_routing_replay=True),
                                   dict(use_rollout_routing_replay=True, use_rollout_logprobs=True)])
@pytest.mark.parametrize("selection", SEL)
def test_teacher_routes_for_itself(selection, flags):
    """With routing replay on, ids and log-probs that reach the loss are those of a teacher that chooses its experts itself, sample by sample
    over several micro-batches; the policy's passes replay what was recorded for them."""
    actor = _actor(selection=selection, **flags)
    batch = _batch(actor, routed="use_rollout_routing_replay" in flags)
    if flags.get("use_rollout_logprobs"):
        batch["rollout_log_probs"] = [[-7.0] * r for r in batch["response_lengths"]]
    seen, made, plain = [], [], actor._distill_ids
    orig = RoutingReplay.route.__func__

    def spy(cls, layer, idx):
        out = orig(cls, layer, idx)
        seen.append((actor._active_tag, cls.mode, bool((out != idx).any())))
        return out

    actor._distill_ids = lambda b: made.append(plain(b)) or made[-1]
    RoutingReplay.route = classmethod(spy)
    try:
        m = actor.train(0, batch)
    finally:
        RoutingReplay.route = classmethod(orig)
    assert RoutingReplay.mode is None and m["opd_loss"] > 0
    assert {mode for tag, mode, _ in seen if tag == "teacher"} == {None}
    assert "replay" in {mode for tag, mode, _ in seen if tag == "actor"}
    ids, _, _, t_lp = made[0]
    for i, (q, lp) in enumerate(_teacher_alone(actor, batch, None if selection == "teacher_topk" else ids)):
        assert torch.equal(ids[i], q)
        there = q >= 0
        # 32-bit logits and their logsumexp against 64-bit ones of the same hidden states, packed differently
        assert torch.allclose(t_lp[i][there].double(), lp[there], atol=1e-4, rtol=0)


def test_policy_passes_on_sets_of_ids_replay_what_was_recorded():
    """The student's own log-probs on its ids come from the experts that the training forward will use, however samples are packed."""
    actor = _actor(use_routing_replay=True)
    batch = _batch(actor)
    RoutingReplay.begin_record()
    want = actor.compute_topk_log_probs(batch, k=5)["ids"]
    kept = dict(RoutingReplay.per_sample)
    assert len(kept) == 4 * sum(actor.mcfg.is_moe_layer(i) for i in range(actor.mcfg.num_layers))
    RoutingReplay.end()
    RoutingReplay.begin_replay()
    for p in actor.model.parameters():      # another router: without replay other experts
        if p.shape == (actor.mcfg.num_experts, actor.mcfg.hidden_size):
            p.data.neg_()
    actor.cfg.micro_batch_size = 3
    calls, orig = [], RoutingReplay.route.__func__

    def spy(cls, layer, idx):
        calls.append(torch.equal(orig(cls, layer, idx), torch.cat([kept[(layer, s)] for s in cls.layout[0]])))
        return orig(cls, layer, idx)

    RoutingReplay.route = classmethod(spy)
    try:
        got = actor.compute_topk_log_probs(batch, ids=want)
    finally:
        RoutingReplay.route = classmethod(orig)
    assert calls and all(calls) and len(got["log_probs"]) == 4


@pytest.mark.parametrize("call", ["compute_log_prob", "compute_topk_log_probs"])
def test_a_failed_teacher_pass_leaves_nothing_behind(call):
    actor = _actor(use_routing_replay=True)
    batch = _batch(actor)
    RoutingReplay.begin_replay()
    actor._pack_batch = lambda *a: (_ for _ in ()).throw(RuntimeError("no room"))
    with pytest.raises(RuntimeError, match="no room"):
        getattr(actor, call)(batch, "teacher", **({"k": 3} if call != "compute_log_prob" else {}))
    assert RoutingReplay.mode == "replay" and actor._active_tag == "actor"


@pytest.mark.parametrize("mode", ["record", "replay"])
def test_a_pass_for_nobody_is_neither_recorded_nor_replayed(mode):
    """A data-parallel rank with fewer micro-batches runs a filler between and after its own."""
    actor = _actor(use_routing_replay=True)
    batch = _batch(actor)
    RoutingReplay.begin_record()
    actor.compute_log_prob(batch)
    kept = dict(RoutingReplay.per_sample)
    RoutingReplay.mode = mode
    actor._dummy_forward()
    actor._dummy_forward(backward=True)
    assert RoutingReplay.per_sample.keys() == kept.keys() and all(RoutingReplay.per_sample[k] is v for k, v in kept.items())


@pytest.mark.parametrize("model,selection", [("tiny", s) for s in SEL] + [("tiny-moe", "union")])
def test_step_trains_on_the_divergence_of_whole_logits(model, selection):
    """A step of pure distillation over several micro-batches: every sample's rows carry its own ids and teacher log-probs, the metric is the
    divergence of whole logits, and parameters get its gradient."""
    from relax_b200.algo import opd

    actor = _actor(model, micro=3, selection=selection, opd_only_reward=True)
    batch = _batch(actor)
    grads, plain = {}, actor.optimizer.step

    def step(**kw):
        for n, p in actor.model.named_parameters():
            grads[n] = (p.grad if p.grad is not None else p.main_grad).detach().clone()
        return plain(**kw)

    made, distill_batch = [], actor._distill_batch
    actor._distill_batch = lambda b, ids: made.append((list(ids), distill_batch(b, ids))) or made[-1][1]
    actor.optimizer.step = step
    m = actor.train(0, batch)
    assert sorted(i for ids, _ in made for i in ids) == [0, 1, 2, 3] and len(made) > 1
    # ids and teacher log-probs of every sample, from the teacher's weights alone
    own = [t for t, _ in _teacher_alone(actor, batch)]
    whole = _teacher_alone(actor, batch, [torch.arange(actor.mcfg.vocab_size).expand(n, -1) for n in batch["response_lengths"]])
    total = 0.0
    model_ = actor.model
    for p in model_.parameters():      # (gradients of their own, apart from the optimizer's buffer)
        p.grad = p.main_grad = None
    for i, (t, r) in enumerate(zip(batch["tokens"], batch["response_lengths"])):
        h = model_(torch.tensor(t), torch.arange(len(t)), torch.tensor([0, len(t)], dtype=torch.int32), max_seqlen=len(t))
        lp = torch.log_softmax(model_.logits(h)[len(t) - r - 1:len(t) - 1, : actor.mcfg.vocab_size].double(), -1)
        student = lp.detach().topk(5, -1).indices
        ids = {"teacher_topk": own[i], "student_topk": student, "union": torch.cat([student, own[i]], 1)}[selection]
        for sids, d in made:
            if i in sids:
                n0 = sum(batch["response_lengths"][s] for s in sids[: sids.index(i)])
                rows = (d["ids"][n0:n0 + r], d["teacher"][n0:n0 + r])
        want_t = whole[i][1]
        for row in range(r):
            got = [int(x) for x in rows[0][row] if x >= 0]
            assert sorted(got) == sorted(set(ids[row].tolist())) and len(got) == len(set(got))
            there = rows[0][row] >= 0
            assert torch.allclose(rows[1][row][there].double(), want_t[row, rows[0][row][there]], atol=1e-4, rtol=0)
        q = rows[0]
        d = opd.token_kl(lp.gather(-1, q.clamp_min(0)), want_t.gather(-1, q.clamp_min(0)).masked_fill(q < 0, 0.0), "jsd", 0.5, "tail", mask=q >= 0)
        total = total + d.mean() / 4
    assert m["opd_loss"] == pytest.approx(float(total), rel=1e-4) and m["pg_loss"] == 0.0
    total.backward()
    ref = {n: (p.grad if p.grad is not None else torch.zeros_like(p)) for n, p in actor.model.named_parameters()}
    norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in ref.values()))
    off = math.sqrt(sum(float((grads[n].double() - ref[n].double()).pow(2).sum()) for n in ref))
    # 32-bit layers on both sides, summed in another order: some thousand roundings of 2^-24
    assert norm > 0 and off <= 1e-3 * norm


def test_what_cannot_be_trained_is_refused_before_anything_is_generated(monkeypatch):
    """Options when they are read, the model's sizes and type when the trainer is made."""
    import dataclasses

    from relax_b200.config.arguments import parse_args

    base = ["--model-name", "tiny", "--colocate", "--rollout-batch-size", "2", "--use-opd", "--opd-teacher-load", "somewhere", "--opd-loss-coef", "1.0",
            "--opd-token-selection", "union", "--opd-log-prob-top-k", "8"]
    assert parse_args(base).opd_loss_coef == 1.0
    for extra, match in ((["--mtp-num-layers", "1"], "multi-token-prediction"), (["--enable-mtp-training"], "multi-token-prediction"),
                         (["--loss-type", "custom_loss", "--custom-loss-function-path", "a.b"], "policy loss"), (["--loss-type", "sft_loss"], "policy loss")):
        with pytest.raises(ValueError, match=match):
            parse_args(base + extra)
        sampled = [x for x in base if x not in ("--opd-token-selection", "union", "--opd-log-prob-top-k", "8")]
        parse_args(sampled + extra)                                   # (the sampled token's term is as it was)
    tiny = get_config("tiny")
    cfg = TrainConfig(opd_token_selection="union", opd_log_prob_top_k=5, loss=LossConfig(opd_loss_coef=1.0))

    class Made(Exception):
        pass

    def no_model(*a, **kw):
        raise Made

    monkeypatch.setattr("relax_b200.train.actor.GPTModel", no_model)      # (nothing of the model is made before the refusal)
    with pytest.raises(NotImplementedError, match="plain decoder"):
        TrainActor(dataclasses.replace(tiny, mtp_num_layers=1), cfg)
    bf = dataclasses.replace(tiny, dtype="bf16")
    for m in (tiny, dataclasses.replace(bf, vocab_size=1020), dataclasses.replace(bf, hidden_size=252)):
        with pytest.raises(ValueError, match="multiples of 8"):
            TrainActor(m, cfg, device="cuda")
        for ok in (dict(device="cuda", role="critic"), dict(device="cpu")):
            with pytest.raises(Made):
                TrainActor(m, cfg, **ok)
    with pytest.raises(Made):
        TrainActor(bf, cfg, device="cuda")


@pytest.mark.parametrize("selection", SEL)
def test_step_reports_finite_numbers(selection):
    """The teacher's log-probs of padded ids (-inf) are no metric."""
    actor = _actor("tiny", selection=selection)
    m = actor.train(0, _batch(actor))
    assert "rollout/opd_teacher_topk_log_probs" not in m and all(math.isfinite(v) for v in m.values() if isinstance(v, (int, float)))


def test_weight_of_the_mixture_is_refused_when_options_are_read():
    from relax_b200.config.arguments import parse_args

    base = ["--model-name", "tiny", "--colocate", "--rollout-batch-size", "2", "--use-opd", "--opd-teacher-load", "somewhere", "--opd-loss-coef", "1.0",
            "--opd-token-selection", "union", "--opd-log-prob-top-k", "8", "--opd-kl-type", "jsd", "--opd-jsd-alpha"]
    for ok in ("0", "0.3", "1"):
        assert parse_args(base + [ok]).opd_jsd_alpha == float(ok)
    for bad in ("-0.1", "1.5", "nan"):
        with pytest.raises(ValueError, match="opd-jsd-alpha"):
            parse_args(base + [bad])


def _two_rank_batch(rows):
    g = torch.Generator().manual_seed(9)
    lens, rl = (30, 28, 11, 9), [7, 9, 4, 3]
    toks = [torch.randint(3, 1000, (n,), generator=g).tolist() for n in lens]
    return {"tokens": [toks[i] for i in rows], "response_lengths": [rl[i] for i in rows], "loss_masks": [[1.0] * rl[i] for i in rows],
            "rewards": [[1.0, 0.0, 0.0, 1.0][i] for i in rows]}


def _two_rank_step(ps, rows, selection):
    """One step on samples ``rows``; the two long ones do not fit one micro-batch, so a rank with the short ones runs a filler."""
    cfg = TrainConfig(advantage_estimator="grpo", global_batch_size=4, n_samples_per_prompt=2, use_dynamic_batch_size=True, max_tokens_per_gpu=32,
                      pad_multiple=1, opd_token_selection=selection, opd_log_prob_top_k=5, opd_kl_type="jsd", opd_only_reward=True, use_routing_replay=True,
                      loss=LossConfig(opd_loss_coef=1.0, opd_kl_type="jsd"), optim=OptimizerConfig(lr=0.0))
    actor = TrainActor(get_config("tiny-moe"), cfg, ps, seed=0)
    teacher = actor.param_buf.clone()
    for p, o in actor._bound_params():      # (the same change of every weight on every rank, however experts are spread)
        teacher[o:o + p.numel()] *= 1.3
    actor.snapshots["teacher"] = teacher
    m = actor.train(0, _two_rank_batch(rows))
    return m["opd_loss"], m["grad_norm"], RoutingReplay.mode


def _two_rank_worker(rank, world, dims, selection):
    from relax_b200.parallel.state import ParallelDims, init_parallel_state

    return _two_rank_step(init_parallel_state(ParallelDims(dp=2, **dims)), [0, 1] if rank == 0 else [2, 3], selection)


@pytest.mark.parametrize("dims,selection", [({}, "union"), ({"ep": 2}, "teacher_topk")])
def test_two_replicas_with_uneven_micro_batches(dims, selection):
    from tests._mp import run_distributed

    got = run_distributed(_two_rank_worker, 2, dims, selection)
    want = _two_rank_step(None, [0, 1, 2, 3], selection)
    assert want[2] is None and want[0] > 0 and want[1] > 0
    for loss, norm, mode in got:      # 32-bit layers, gradients summed in another order
        assert mode is None and loss == pytest.approx(want[0], rel=1e-4) and norm == pytest.approx(want[1], rel=1e-3)
