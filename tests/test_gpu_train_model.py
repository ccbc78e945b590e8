"""The operators of a training step together: GPT's embeddings and dropout, graphs, streams, and the example that tunes."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tests.block_helpers import close
from tests.train_helpers import factors

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "isa-_amd" / "examples"))


def make_gpt(dev, dropout=0.0, layers=2, dim=48, vocab=70, positions=40):
    from isa.operators.block import GPT, Block, WindowAttention

    torch.manual_seed(0)
    blocks = nn.ModuleList(Block(dim, WindowAttention(dim, 3, window=9, sinks=2), nn.Linear(dim, dim), dropout)
                           for _ in range(layers))
    return GPT(vocab, positions, dim, blocks, dropout).to(dev)


def plain_gpt(model, ids, masks):
    """GPT.forward of torch's embeddings and sums, with masks [site] of factors, and the model's own attention and norms."""
    def drop(site, t):
        return t if masks is None else t * masks[site].view(t.shape)

    x = drop(0, F.embedding(ids, model.tokens.weight) + model.positions.weight[: ids.shape[1]])
    for i, block in enumerate(model.blocks):
        if i:
            x = x + drop(1 + 2 * i, branch)
        x = x + drop(2 + 2 * i, block.attention(F.layer_norm(x, x.shape[-1:], block.ln1.weight, block.ln1.bias)))
        branch = block.ffn(F.layer_norm(x, x.shape[-1:], block.ln2.weight, block.ln2.bias))
    x = x + drop(1 + 2 * len(model.blocks), branch)
    return F.linear(F.layer_norm(x, x.shape[-1:], model.ln_f.weight, model.ln_f.bias), model.tokens.weight)


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_gpt_matches_torch(cuda_device, p):
    """fp32 in two orders of summation: some 100 roundings of 2^-24."""
    from isa.operators.block import DropoutSeed

    model = make_gpt(cuda_device, p)
    ids = torch.randint(0, 70, (3, 25), device=cuda_device)
    up = torch.randn(3, 25, 70, device=cuda_device)
    if p:
        model.seed = DropoutSeed(key=77)
    got = model(ids)
    grads = torch.autograd.grad(got, list(model.parameters()), up)
    masks = None
    if p:
        assert model.seed.state.tolist() == [77, 6]  # past its sites
        masks = [factors(75, 48, p, (77, 0), site).float().to(cuda_device) for site in range(6)]
    want = plain_gpt(model, ids, masks)
    close(got, want, 2e-5, "logits")
    for a, b, (name, _) in zip(grads, torch.autograd.grad(want, list(model.parameters()), up), model.named_parameters()):
        close(a, b, 3e-5, name)
    model.eval()
    close(model(ids), plain_gpt(model, ids, None), 2e-5, "evaluation")


def test_state_dict_and_seeds(cuda_device):
    from isa.operators.block import Embedding

    a, b = make_gpt(cuda_device, 0.1), make_gpt(cuda_device)
    assert list(a.state_dict()) == list(b.state_dict()) and all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))
    ids = torch.randint(0, 70, (2, 10), device=cuda_device)
    first, second = a(ids), a(ids)
    assert not torch.equal(first, second)  # another step, other numbers
    a.seed.state[1] = 0
    assert torch.equal(a(ids), first)
    theirs, ours = nn.Embedding(20, 12, padding_idx=3).to(cuda_device), Embedding(20, 12, padding_idx=3).to(cuda_device)
    ours.load_state_dict(theirs.state_dict())
    x = torch.randint(0, 20, (4, 30), device=cuda_device)
    assert torch.equal(ours(x), theirs(x))
    up = torch.randn(4, 30, 12, device=cuda_device)
    close(torch.autograd.grad(ours(x), ours.weight, up)[0], torch.autograd.grad(theirs(x), theirs.weight, up)[0], 2e-6, "dweight")
    for option in ({"max_norm": 1.0}, {"scale_grad_by_freq": True}, {"sparse": True}):
        with pytest.raises(ValueError, match="not supported"):
            Embedding(4, 4, **option)
    # a caller's own tables
    b.positions = nn.Embedding.from_pretrained(b.positions.weight.detach().clone()).to(cuda_device)
    assert torch.equal(b(ids), make_gpt(cuda_device)(ids))


def test_a_captured_step_draws_anew(cuda_device):
    """A training step of all operators as a graph: every replay equals the eager step of the same seed, with other work
    and synchronisations between replays."""
    from isa.kernels.transformer_block import policy_loss_with_grad
    from isa.operators.block import DropoutSeed

    model = make_gpt(cuda_device, 0.2)
    params = list(model.parameters())
    g = torch.Generator(device=cuda_device).manual_seed(1)
    ids = torch.randint(0, 70, (4, 20), generator=g, device=cuda_device)
    actions = torch.randint(0, 70, (4, 20), generator=g, device=cuda_device)
    old = torch.full((4, 20), -4.0, device=cuda_device)
    advantages = torch.randn(4, 20, generator=g, device=cuda_device)

    def step():
        logits = model(ids)
        loss, gradient, logp = policy_loss_with_grad(logits, actions, old, advantages, kl=0.1, ref_logp=old)
        return [loss, logp, *torch.autograd.grad(logits, params, gradient)]

    model.seed = DropoutSeed(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        ids.copy_(torch.randint(0, 70, ids.shape, generator=g, device=cuda_device))
        before = model.seed.state.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert model.seed.state.tolist() == [5, int(before[1]) + 6]
        got = [t.clone() for t in out]
        model.seed.state.copy_(before)
        want = step()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (turn, i)
        del want
        torch.randn(1000, 1000, device=cuda_device).sum().item()


def test_capture_beside_a_living_graph_is_refused(cuda_device):
    """A leaf whose accumulator was made on the default stream cannot take part in a capture."""
    from isa.kernels.transformer_block import dropout, dropout_add_layer_norm, embedding, policy_loss, preference_loss

    dev = cuda_device
    seed = torch.tensor([1, 2], device=dev)
    w = torch.randn(10, 16, device=dev, requires_grad=True)
    one = torch.ones(16, device=dev)
    ids = torch.randint(0, 10, (4,), device=dev)
    f = torch.zeros(10, device=dev)
    x3 = torch.randn(2, 3, 8, device=dev, requires_grad=True)
    t, t2 = torch.zeros(10, dtype=torch.int64, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev)
    calls = {"embedding": (w, lambda: embedding(ids, w)), "dropout": (w, lambda: dropout(w, 0.5, seed)),
             "norm": (w, lambda: dropout_add_layer_norm(w, w, one, p=0.5, seed=seed)),
             "policy": (w, lambda: policy_loss(w, t, f, f)), "preference": (x3, lambda: preference_loss(x3, t2, f[:2]))}
    for name, (leaf, call) in calls.items():
        print(f"[case] {name}", flush=True)
        call()
        living = (leaf * 2.0)  # its accumulator is made here
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        refused = []
        inputs = torch.zeros(4, device=dev)
        with torch.cuda.graph(graph):
            try:
                call()
            except RuntimeError as e:
                refused.append(str(e))
            inputs.add_(1.0)
        assert len(refused) == 1 and "before a step with that leaf is captured" in refused[0], refused
        graph.replay()
        torch.cuda.synchronize()
        assert float(inputs[0]) == 1.0
        del living


def test_two_streams(cuda_device):
    """Calls on two streams at once, each with its own workspace, give what they give alone."""
    from isa.kernels.transformer_block import embedding, policy_loss_with_grad, preference_loss_with_grad

    g = torch.Generator(device=cuda_device).manual_seed(0)
    sets = []
    for k in range(2):
        ids = torch.randint(0, 300, (9000,), generator=g, device=cuda_device)
        ids[: 3000 * (k + 1)] = k
        w = torch.randn(300, 64, generator=g, device=cuda_device, requires_grad=True)
        dy = torch.randn(9000, 64, generator=g, device=cuda_device)
        x = torch.randn(64, 32, 500, generator=g, device=cuda_device)
        t = torch.randint(0, 500, (64, 32), generator=g, device=cuda_device)
        f = torch.randn(64, 32, generator=g, device=cuda_device)
        sets.append((ids, w, dy, x, t, f))

    def run(ids, w, dy, x, t, f):
        return [torch.autograd.grad(embedding(ids, w), w, dy)[0], *policy_loss_with_grad(x, t, f - 6.0, f),
                *preference_loss_with_grad(x, t, f[:, 0] - 200.0)]

    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(run(*s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_example_tunes(cuda_device):
    """It runs, its ratios are 1 before a step (the loss is the rewards' mean, near 0), and its gradients are torch's."""
    import copy

    import tune_window_gpt as example
    from isa.kernels.transformer_block import preference_loss_with_grad

    torch.manual_seed(0)
    generator = torch.Generator(device="cuda").manual_seed(0)
    model = example.make_model(dropout=0.05)
    example.train(model, 5, generator)
    model.eval()
    reference = copy.deepcopy(model).requires_grad_(False)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-4)
    reward, losses = example.policy_step(model, reference, optimizer, generator)
    assert 0.0 <= reward <= 1.0 and abs(losses[0]) <= 1e-4 and all(x == x for x in losses)
    assert example.preference_step(model, reference, optimizer, generator) > 0.0
    # the gradients that tune it, against torch's of the same loss
    ids = example.batch(6, 30, generator)
    targets = example.targets_of(ids)
    logits = model(ids).detach()
    _, gradient, _ = preference_loss_with_grad(logits, targets, torch.zeros(6, device=cuda_device), beta=0.05)
    leaf = logits.double().requires_grad_(True)
    nll = F.cross_entropy(leaf.view(-1, leaf.shape[-1]), targets.view(-1), ignore_index=-100, reduction="none")
    total = -nll.view(6, 30).sum(1)
    (want,) = torch.autograd.grad(-F.logsigmoid(0.05 * (total[:3] - total[3:])).mean(), leaf)
    close(gradient, want, 1e-5, "gradient")
