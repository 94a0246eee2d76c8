"""The vocabulary operators as a user runs them together: a teacher policy's record, a student's distillation step and
training loop, and decoding from filtered distributions with the vocabulary matrix in float32 or 8 bits.  Needs an MI355X."""
import importlib

import numpy as np
import pytest
import torch

from helpers import synthetic
from oracle import vocab_refs as ref

pytestmark = pytest.mark.gpu

hip = importlib.import_module("image-captioning-through-rl_amd.hipabi")
models = importlib.import_module("image-captioning-through-rl_amd.models")
trainers = importlib.import_module("image-captioning-through-rl_amd.trainers")
engine_mod = importlib.import_module("image-captioning-through-rl_amd.engine")


def policy(vocab, fdim, seed):
    net = models.PolicyNetwork(synthetic.make_word_to_idx(vocab), input_dim=fdim)
    net.load_state_dict({k: torch.from_numpy(v.copy()) for k, v in synthetic.make_params("policy", vocab, fdim, seed).items()})
    return net.cuda()


def double_logits(net, features, captions):
    """The policy network's logits [L, N, V] in float64 on the CPU, with a graph to its parameters."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in net.named_parameters()}
    n, length = captions.shape
    h = features.double().cpu() @ p["cnn2linear.weight"].t() + p["cnn2linear.bias"]
    c = torch.zeros(n, 512, dtype=torch.float64)
    out = []
    for t in range(length):
        x = p["caption_embedding.weight"][captions[:, t].cpu()]
        gates = x @ p["lstm.weight_ih_l0"].t() + p["lstm.bias_ih_l0"] + h @ p["lstm.weight_hh_l0"].t() + p["lstm.bias_hh_l0"]
        i, f, g, o = gates.split(512, dim=1)
        c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(g)
        h = torch.sigmoid(o) * torch.tanh(c)
        out.append(h @ p["linear2vocab.weight"].t() + p["linear2vocab.bias"])
    return torch.stack(out), p


@pytest.mark.parametrize("vocab,n,length,top,tail", [(100, 5, 6, 8, True), (257, 12, 9, 32, True), (300, 4, 5, 16, False)])
@pytest.mark.parametrize("grad_products", ["f32", "f16x2"])
def test_distillation_step_against_float64_autograd(vocab, n, length, top, tail, grad_products):
    fdim, temp = 512, 1.5
    features, captions = synthetic.make_minibatch(n, vocab, length, fdim, 3)
    feats, caps = torch.from_numpy(features).cuda(), torch.from_numpy(captions).cuda()
    teacher, student = policy(vocab, fdim, 1), policy(vocab, fdim, 2)
    values, indices, lse = trainers.teacher_record(teacher, feats, caps, top, temp)
    weight = torch.rand(length - 1, n, generator=torch.Generator().manual_seed(0)).cuda()
    weight[-1, ::2] = 0.0
    grads = {k: torch.full_like(v, 7.0) for k, v in student.named_parameters()}
    engine = engine_mod.A2CEngine({k: v.data for k, v in student.named_parameters()}, None, None, grads, grad_products=grad_products)
    loss = engine.policy_distill_step(feats, caps, (values, indices, lse if tail else None), weight, temp).item()

    # the record is the teacher's
    t_logits = double_logits(teacher, feats, caps[:, :-1])[0].reshape(-1, vocab).detach().numpy()
    for r in range(t_logits.shape[0]):
        want_v, _, want_l = ref.topk_lse(t_logits[r], top, temp)
        assert np.abs(values[r].cpu().numpy() - want_v).max() < 2e-5 and abs(lse[r].item() - want_l) < 2e-5
    # loss and gradients by automatic differentiation in float64
    logits, p = double_logits(student, feats, caps[:, :-1])
    z = logits.reshape(-1, vocab) / temp
    log_p = torch.log_softmax(z, 1)
    log_q = values.double().cpu() / temp
    log_q = log_q - lse.double().cpu().view(-1, 1) if tail else torch.log_softmax(log_q, 1)
    q = log_q.exp()
    rows = (q * (log_q - log_p.gather(1, indices.cpu()))).sum(1)
    if tail:
        left = 1.0 - q.sum(1)
        rest = torch.ones_like(log_p).scatter(1, indices.cpu(), 0.0)
        rows = rows + left * (left.log() - (log_p.exp() * rest).sum(1).log())
    want = (rows * weight.reshape(-1).double().cpu()).sum()
    want.backward()
    assert abs(loss - want.item()) <= 2e-5 * abs(want.item())
    for k, g in grads.items():
        w = p[k].grad
        # float32 sums over all positions and back through the recurrence: relative to each tensor's norm
        assert (g.double().cpu() - w).norm() <= 2e-5 * w.norm() + 1e-9, (k, float((g.double().cpu() - w).norm() / w.norm()))


def test_a_student_learns_its_teachers_distribution(tmp_path):
    """The training loop runs, saves, logs, and leaves an A2C or cross-entropy step of the same engine shape untouched."""
    n, vocab, fdim = 8, 60, 512
    data = synthetic.make_ragged_train_data(n, vocab, fdim, 4, max_len=9)
    log = trainers.ScalarLog()
    paths = {"policy_network": str(tmp_path / "student.pt")}
    torch.manual_seed(0)
    student = trainers.distill_policy_network(data, policy(vocab, fdim, 5), paths, log, epochs=3, batch_size=n, top=10)
    values = [v for tag, v, _ in log.records if tag == "Policy Network-distillation-loss"]
    assert len(values) == 3 and all(np.isfinite(values))
    saved = torch.load(paths["policy_network"], map_location="cuda", weights_only=True)
    assert saved.keys() == student.state_dict().keys()


def test_distillation_step_leaves_other_steps_alone():
    n, vocab, fdim, length = 6, 200, 512, 7
    features, captions = synthetic.make_minibatch(n, vocab, length, fdim, 6)
    feats, caps = torch.from_numpy(features).cuda(), torch.from_numpy(captions).cuda()
    net = policy(vocab, fdim, 7)
    grads = {k: torch.zeros_like(v) for k, v in net.named_parameters()}
    engine = engine_mod.A2CEngine({k: v.data for k, v in net.named_parameters()}, None, None, grads)
    valid = torch.full((n,), length - 1, dtype=torch.int32, device="cuda")
    weight = torch.full((n,), 1.0 / n, device="cuda")
    loss = engine.policy_ce_step(feats, caps, valid, weight).clone()
    first = {k: g.clone() for k, g in grads.items()}
    record = trainers.teacher_record(policy(vocab, fdim, 8), feats, caps, 20, 2.0)
    engine.policy_distill_step(feats, caps, record, torch.ones(length - 1, n, device="cuda"), 2.0)
    distilled = {k: g.clone() for k, g in grads.items()}
    again = engine.policy_ce_step(feats, caps, valid, weight)
    assert torch.equal(loss, again) and all(torch.equal(first[k], grads[k]) for k in grads)
    engine.policy_distill_step(feats, caps, record, torch.ones(length - 1, n, device="cuda"), 2.0)
    assert all(torch.equal(distilled[k], grads[k]) for k in grads)


def test_sampled_decoding_against_the_reference_draws():
    n, vocab, fdim = 7, 300, 512
    net = policy(vocab, fdim, 9)
    features = torch.from_numpy(synthetic.make_minibatch(n, vocab, 6, fdim, 10)[0]).cuda()
    start = torch.ones(n, 1, dtype=torch.int64, device="cuda")
    u = np.random.RandomState(11).random_sample((16, n))
    temperature = torch.tensor([0.0, 0.5, 1.0, 1.0, 2.0, 1.0, 0.7], device="cuda")
    settings = dict(temperature=temperature, top_k=40, top_p=0.9, min_p=0.01)
    tokens, log_prob = trainers.GenerateCaptionsSampled(features, start, net, uniforms=torch.from_numpy(u), **settings)
    assert tokens.shape == (n, 17) and log_prob.shape == (n, 16)
    logits = net(features.unsqueeze(0), tokens[:, :-1]).cpu().double().numpy()
    for i in range(n):
        for t in range(16):
            tok, lp = ref.sample_filtered(logits[i, t], u[t, i], float(temperature[i]), 40, 0.9, 0.01)
            assert tokens[i, t + 1].item() == tok and abs(log_prob[i, t].item() - lp) < 1e-4
    greedy = trainers.GenerateCaptionsGreedy(features, start, net)
    assert torch.equal(greedy, trainers.GenerateCaptionsSampled(features, start, net, temperature=0.0)[0])
    np.random.seed(3)
    a = trainers.GenerateCaptionsSampled(features, start, net)[0]
    np.random.seed(3)
    assert torch.equal(a, trainers.GenerateCaptionsSampled(features, start, net)[0])


def test_sampled_decoding_refuses_a_row_that_cannot_draw():
    net = policy(120, 512, 12)
    features = torch.zeros(3, 512, device="cuda")
    start = torch.ones(3, 1, dtype=torch.int64, device="cuda")
    bad = torch.tensor([1.0, -1.0, 1.0], device="cuda")
    with pytest.raises(RuntimeError, match="row 1"):
        trainers.GenerateCaptionsSampled(features, start, net, temperature=bad)
    with pytest.raises(AssertionError):
        trainers.GenerateCaptionsSampled(features, start, net, uniforms=torch.zeros(16, 4, dtype=torch.float64))


@pytest.mark.parametrize("n", [1, 5, 70])
def test_decoding_with_the_eight_bit_vocabulary_matrix(n):
    vocab, fdim = 500, 512
    net = policy(vocab, fdim, 13)
    features = torch.from_numpy(synthetic.make_minibatch(n, vocab, 6, fdim, 14)[0]).cuda()
    start = torch.ones(n, 1, dtype=torch.int64, device="cuda")
    tokens, _ = trainers.GenerateCaptionsSampled(features, start, net, temperature=0.0, vocab8=net.vocab_weight8())
    logits = net(features.unsqueeze(0), tokens[:, :-1])
    # both operands are rounded by at most 2^-4 of themselves (or 2^-10 of a scale that is at most 2 / 448 of the block's
    # largest), |h| < 1: a logit is off by at most this, so the chosen word's is within twice that of the largest
    w = net.linear2vocab.weight.abs()
    off = ((2.0 ** -3 + 2.0 ** -8) * w.sum(1) + 512 * 2.0 ** -10 / 224 * (w.max(1).values + 1.0) + 1e-4).max()
    chosen = logits.gather(2, tokens[:, 1:].unsqueeze(2)).squeeze(2)
    assert (chosen >= logits.max(2).values - 2 * off).all()


def test_a_teachers_record_of_a_small_vocabulary_holds_all_of_it():
    net = policy(40, 32, 3)
    feats = torch.randn(4, 32, generator=torch.Generator().manual_seed(9)).cuda()
    caps = torch.randint(0, 40, (4, 6), generator=torch.Generator().manual_seed(10)).cuda()
    values, indices, lse = trainers.teacher_record(net, feats, caps, 64, 1.5)
    assert values.shape == indices.shape == (20, 40) and lse.shape == (20,)
    assert torch.equal(indices.sort(dim=1).values, torch.arange(40, device="cuda").expand(20, 40))
    # the values are exact copies; float64 on the CPU sums them, so that the record's float32 is off by its own rounding, and
    # by the 40 float32 exponentials' (2^-22 of the sum at most, each one's argument and result together)
    want = torch.logsumexp(values.double().cpu() / 1.5, dim=1)
    assert (lse.double().cpu() - want).abs().max() <= 2.0 ** -22 + 2.0 ** -24 * float(want.abs().max())
