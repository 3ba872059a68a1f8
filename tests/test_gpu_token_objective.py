"""A per-token objective from tokens to updated weights: GemmaTextModel.token_logprobs, the caller's loss, the backward
of everything, AdamW with the global norm's clipping."""
import copy

import pytest
import torch

from maester_amd import AdamW, token_logprobs
from maester_amd.gemma_layers import GemmaLayerConfig, GemmaTextModel
from maester_amd.packed_ids import packed_collate_ids

pytestmark = pytest.mark.gpu
B, S = 2, 290


def setup(gpu):
    torch.manual_seed(3)
    cfg = GemmaLayerConfig(dim=256, n_heads=4, num_key_value_heads=2, head_dim=128, max_seq_len=512, sliding_window_size=64,
                           intermediate_size=512, n_layers=2, attn_types=("local_sliding", "global"), vocab_size=1003)
    rows = [[(0, 0, 90), (1, 90, 200)], [(2, 0, 150), (3, 150, 100)]]
    pos, doc = (x.to(gpu) for x in packed_collate_ids(rows, S))
    model = GemmaTextModel(cfg).to(gpu).to(torch.bfloat16)
    model.init_weights(0.06)
    tokens = torch.randint(0, cfg.vocab_size, (B, S), device=gpu)
    labels = torch.roll(tokens, -1, 1)
    labels[:, :40] = -100
    labels[doc < 0] = -100
    advantage = torch.randn(B, S, device=gpu)
    return model, tokens, labels, pos, doc, advantage


def objective(logp, entropy, advantage, labels):
    keep = (labels != -100).sum()
    return -(advantage * logp).sum() / keep - 0.01 * entropy.sum() / keep


def test_model_scores_tokens(gpu):
    # against the log-softmax of the model's own bf16 logits: those carry a rounding of 2^-9 of values up to about 10
    model, tokens, labels, pos, doc, advantage = setup(gpu)
    logp, entropy = model.token_logprobs(tokens, labels, pos, doc)
    assert logp.shape == (B, S) and logp.dtype == torch.float32 and torch.all(logp[labels == -100] == 0)
    x = model(tokens, None, pos, doc)
    tol = 2 * 2.0 ** -8 * float(x.abs().max())
    want = token_logprobs(x, labels)
    assert float((logp - want.logp).abs().max()) <= tol and float((entropy - want.entropy).abs().max()) <= 4 * tol
    # the mean negative log-probability is the model's loss
    loss = model(tokens, labels, pos, doc)
    assert abs(float(-logp.sum() / (labels != -100).sum()) - float(loss)) <= tol
    # both forms lead to the same gradients of the weights, up to the roundings of the logits and their gradient
    grads = []
    for form in (lambda: model.token_logprobs(tokens, labels, pos, doc), lambda: token_logprobs(model(tokens, None, pos, doc), labels)[:2]):
        model.zero_grad()
        objective(*form(), advantage, labels).backward()
        grads.append([p.grad.float().clone() for p in model.parameters()])
    for a, b in zip(*grads):
        assert torch.isfinite(a).all() and float((a - b).norm()) <= 3e-2 * float(b.norm()) + 1e-6


@pytest.mark.parametrize("state_bits,master", [(32, True), (8, True), (8, False)])
def test_steps_of_the_whole(gpu, state_bits, master):
    model, tokens, labels, pos, doc, advantage = setup(gpu)
    opt = AdamW(model.parameters(), lr=1e-3, state_bits=state_bits, master_weights=master, max_grad_norm=0.5)
    # torch's update of fp32 copies from the very gradients that the step saw
    twin = [p.detach().float().clone().requires_grad_() for p in model.parameters()]
    ref = torch.optim.AdamW(twin, lr=1e-3, foreach=False)
    for step in range(2):
        opt.zero_grad()
        objective(*model.token_logprobs(tokens, labels, pos, doc), advantage, labels).backward()
        for t, p in zip(twin, model.parameters()):
            t.grad = p.grad.float()
        norm = torch.nn.utils.clip_grad_norm_(twin, 0.5)
        opt.step()
        ref.step()
        assert abs(float(opt.grad_norm) - float(norm)) <= 1e-5 * float(norm)
        for t, p in zip(twin, model.parameters()):
            # the first step takes its moments from the gradient itself; the second from states in 8 bits where asked: each of
            # m and sqrt(v) a code (2^-3) off at most, of an update of at most the rate each step
            slack = 1e-3 * (1e-3 if state_bits == 32 or step == 0 else 0.6) + 1e-6
            held = opt.state[p]["master"] if master else p.float()
            rounding = 0.0 if master else (step + 1) * 2.0 ** -8
            # (m / (sqrt(v) + eps) of gradients far below eps turns on the last bits of the clipping)
            assert bool(((held - t).abs() <= slack + 2e-5 + rounding * t.abs()).all()), (step, float((held - t).abs().max()))
            if master:
                assert torch.equal(p, held.bfloat16())
                with torch.no_grad():
                    t.copy_(held)
    again = copy.deepcopy(opt.state_dict())
    assert set(again["state"][0]) == {"exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if state_bits == 8 else set()) | ({"master"} if master else set())


def test_training_step_in_a_graph(gpu):
    # scoring, loss, backward and update captured once and replayed: as eager steps, bit for bit
    model, tokens, labels, pos, doc, advantage = setup(gpu)
    twin = copy.deepcopy(model)
    h = {}
    for name, net in (("graph", model), ("eager", twin)):
        with torch.no_grad():
            hidden = net._hidden_states(tokens, pos, doc).clone()
        w = net.tok_embeddings.weight.detach().clone().requires_grad_()
        h[name] = (hidden, w, AdamW([w], lr=1e-2, state_bits=8, max_grad_norm=1.0))

    def step(name):
        from maester_amd import linear_token_logprobs
        hidden, w, opt = h[name]
        logp, entropy = linear_token_logprobs(hidden, w, labels, filter_ignored=False)
        w.grad = torch.autograd.grad(objective(logp, entropy, advantage, labels), w)[0]
        opt.step()
        return logp.detach()

    for name in h:
        step(name)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step("graph")
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = step("eager")
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(h["graph"][1], h["eager"][1]), i
