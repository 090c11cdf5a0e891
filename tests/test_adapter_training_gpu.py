"""Adapters inside a training step: the autograd nodes against fp64, against differences, chunked, captured, and a rollout with
drafted tokens whose log-probabilities the update then reproduces.  Needs an MI355X."""
import pytest
import torch
import torch.nn.functional as F

from oracle import lora_ref, verify_ref
from oracle import logprob_ref as O
from rl_engine.kernels.autograd import lora_linear, lora_linear_logp

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _model(n, h, v, r, s, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda std, *shape: (torch.randn(*shape, generator=g) * std).to(dtype)  # noqa: E731
    return dict(hidden=rnd(1.0, n, h), weight=rnd(h ** -0.5, v, h), a=rnd(h ** -0.5, s, r, h), b=rnd(0.3, s, v, r),
                ids=torch.randint(-1, s, (n,), generator=g), tokens=torch.randint(0, v, (n,), generator=g),
                scaling=torch.rand(s, generator=g) + 0.5, grad=torch.randn(n, generator=g))


def _leaves(c, *names):
    return [c[k].cuda().requires_grad_(True) for k in names]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead", [(70,), (2, 5, 7)])
def test_lora_linear_node(sampler, dtype, lead):
    """Every gradient of the node, element by element within the bounds of the operator's oracle."""
    c = _model(70, 96, 200, 12, 4, dtype, seed=3)
    g = torch.Generator().manual_seed(4)
    base, dy = (torch.randn(70, 200, generator=g).to(dtype) for _ in range(2))
    basex = base.cuda().view(*lead, -1).requires_grad_(True)
    hx = c["hidden"].cuda().view(*lead, -1).requires_grad_(True)
    ax, bx = _leaves(c, "a", "b")
    ids, scaling = c["ids"].cuda().view(lead), c["scaling"].cuda()
    out = lora_linear(sampler, basex, hx, ax, bx, ids, scaling)
    assert out.shape == (*lead, 200) and out.requires_grad
    out.backward(dy.cuda().view(*lead, -1))
    y, _, bound, _ = lora_ref.forward(base, c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    assert ((out.detach().cpu().double().view(70, -1) - y).abs() <= bound).all()
    assert torch.equal(basex.grad.cpu().view(70, -1), dy)
    _, u = sampler.lora_linear(basex.detach(), hx.detach(), ax.detach(), bx.detach(), ids, scaling, return_shrunk=True)
    want, bounds = lora_ref.backward(dy, c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], u.cpu().view(70, -1), None)
    half = torch.finfo(dtype).eps / 2
    assert ((hx.grad.cpu().double().view(70, -1) - want[0]).abs() <= bounds[0]).all()
    for got, w, e in ((ax.grad, want[1], bounds[1]), (bx.grad, want[2], bounds[2])):  # rounded to the parameters' type
        tiny = torch.finfo(dtype).tiny * half
        assert got.dtype == dtype and ((got.cpu().double() - w).abs() <= e + half * (w.abs() + e) + tiny).all()


def test_only_the_gradients_asked_for(sampler):
    c = _model(9, 64, 40, 8, 2, torch.bfloat16, seed=5)
    base = torch.randn(9, 40, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    h, a, b = (c[k].cuda() for k in ("hidden", "a", "b"))
    out = lora_linear(sampler, base, h, a, b, c["ids"].cuda(), 2.0)
    out.float().sum().backward()
    assert torch.equal(base.grad, torch.ones_like(base))
    b.requires_grad_(True)
    lora_linear(sampler, base.detach(), h, a, b, c["ids"].cuda(), 2.0).float().sum().backward()
    assert b.grad is not None and a.grad is None and h.grad is None


@pytest.mark.parametrize("which", ["a", "b", "hidden"])
def test_gradients_against_differences(sampler, which):
    """out is linear in each of its inputs, so L(x1) - L(x2) = <dL/dx, x1 - x2> for L = <w, out> exactly; w is chosen along the
    difference of the outputs, so that rounding (half a step of every output, counted in full) stays far below it."""
    c = _model(33, 128, 72, 16, 3, torch.bfloat16, seed=6)
    g = torch.Generator().manual_seed(7)
    other = (torch.randn(c[which].shape, generator=g) * c[which].double().std()).to(torch.bfloat16)
    base = torch.zeros(33, 72, dtype=torch.bfloat16)

    def run(x):
        t = {k: (x if k == which else c[k]).cuda() for k in ("hidden", "a", "b")}
        t[which].requires_grad_(True)
        return lora_linear(sampler, base.cuda(), t["hidden"], t["a"], t["b"], c["ids"].cuda(), c["scaling"].cuda()), t[which]

    out1, leaf = run(c[which])
    out2, _ = run(other)
    w = (out1 - out2).detach()
    out1.backward(w)
    left = (w.double() * (out1.detach().double() - out2.detach().double())).sum().item()
    right = (leaf.grad.double().cpu() * (c[which].double() - other.double())).sum().item()
    rounding = 2.0 ** -8 * ((w.double().abs() * (out1.detach().double().abs() + out2.detach().double().abs())).sum().item()
                            + (leaf.grad.double().cpu().abs() * (c[which].double() - other.double()).abs()).sum().item())
    rounding *= 1.0 + 2.0 ** -6  # what the fp32 sums and u's 17 bits add is below a hundredth of bf16's half step
    assert rounding < 0.25 * abs(left)
    assert abs(left - right) <= rounding


def _exact_logp(c):
    x, w, a, b = (c[k].double() for k in ("hidden", "weight", "a", "b"))
    x, a, b = (t.clone().requires_grad_(True) for t in (x, a, b))
    ids = c["ids"]
    logits = x @ w.t()
    on = (ids >= 0).double() * c["scaling"].double()[ids.clamp(min=0)]
    u = (a[ids.clamp(min=0)] @ x.unsqueeze(2)) * on.view(-1, 1, 1)
    logits = logits + (b[ids.clamp(min=0)] @ u).squeeze(2)
    logp = torch.log_softmax(logits, -1).gather(1, c["tokens"][:, None]).squeeze(1)
    logp.backward(c["grad"].double())
    return logits.detach(), logp.detach(), x.grad, a.grad, b.grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunk", [None, 20])
def test_lora_linear_logp_against_fp64(sampler, dtype, chunk):
    """The frozen head's logits are rounded twice (product, then product + adapter), so a log-probability is off by at most
    twice two half steps of the largest logit; the gradients carry the rounding of the logit gradients (one half step and what
    the logits' rounding does to a softmax, twice two half steps of the largest logit) and of the result: by relative norm."""
    c = _model(61, 128, 1000, 16, 3, dtype, seed=8)
    hx, ax, bx = _leaves(c, "hidden", "a", "b")
    logp = lora_linear_logp(sampler, hx, c["weight"].cuda(), ax, bx, c["tokens"].cuda(), c["ids"].cuda(), c["scaling"].cuda(),
                            chunk_tokens=chunk)
    (logp * c["grad"].cuda()).sum().backward()
    logits, want, dx, da, db = _exact_logp(c)
    half, top = torch.finfo(dtype).eps / 2, logits.abs().max().item()
    base_top = (c["hidden"].double() @ c["weight"].double().t()).abs().max().item()
    shift = 2 * half * (top + base_top) + 1e-5
    assert (logp.detach().cpu().double() - want).abs().max().item() <= shift
    for got, w in ((hx.grad, dx), (ax.grad, da), (bx.grad, db)):
        assert got.dtype == dtype
        assert ((got.cpu().double() - w).norm() / w.norm()).item() <= shift + 3 * half


def test_lora_linear_logp_chunks_and_no_adapter(sampler):
    """Without adapters it is the frozen head alone; an empty batch has no rows and zero gradients."""
    c = _model(50, 64, 136, 8, 2, torch.bfloat16, seed=9)
    none = torch.full((50,), -1, device="cuda")
    hx, ax, bx = _leaves(c, "hidden", "a", "b")
    logp = lora_linear_logp(sampler, hx, c["weight"].cuda(), ax, bx, c["tokens"].cuda(), none)
    logp.sum().backward()
    want = sampler.compute_logp(F.linear(hx.detach(), c["weight"].cuda()), c["tokens"].cuda())
    assert torch.equal(logp.detach(), want)
    assert not ax.grad.any() and not bx.grad.any() and hx.grad.any()
    empty = lora_linear_logp(sampler, hx[:0], c["weight"].cuda(), ax, bx, c["tokens"][:0].cuda(), none[:0])
    assert empty.shape == (0,)
    ax.grad = None
    empty.sum().backward()
    assert not ax.grad.any()


def test_training_step_replayed_from_a_hip_graph(sampler):
    """Forward and backward of the node captured together: every replay on new inputs gives the eager bits."""
    c = _model(40, 96, 264, 16, 3, torch.bfloat16, seed=10)
    static = {k: c[k].cuda() for k in ("hidden", "a", "b", "ids", "scaling")}
    base, dy = (torch.randn(40, 264, device="cuda").bfloat16() for _ in range(2))

    def step():
        leaves = [static[k].detach().requires_grad_(True) for k in ("hidden", "a", "b")]
        out = lora_linear(sampler, base, *leaves, static["ids"], static["scaling"])
        return (out.detach(), *torch.autograd.grad(out, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    g = torch.Generator().manual_seed(11)
    for _ in range(3):
        static["hidden"].copy_(torch.randn(40, 96, generator=g).cuda())
        static["ids"].copy_(torch.randint(-1, 3, (40,), generator=g).cuda())
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


class _Policy:
    """A toy model: the state behind a token is a row of a table; a shared head, and an adapter per request."""

    def __init__(self, sampler, h, v, r, adapters, seed, k):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda std, *shape: (torch.randn(*shape, generator=g) * std).bfloat16().cuda()  # noqa: E731
        self.sampler, self.k = sampler, k
        self.states, self.head = rnd(1.0, v, h), rnd(3.0 * h ** -0.5, v, h)
        self.a, self.b = rnd(h ** -0.5, 3, r, h), rnd(0.5, 3, v, r)
        self.adapters = adapters.cuda()
        self.log = []

    def logits(self, tokens):
        x = self.states[tokens]
        return self.sampler.lora_linear(F.linear(x, self.head), x, self.a, self.b,
                                        self.adapters[:, None].expand(tokens.shape).contiguous(), 1.5)

    def propose(self, ids, lengths):
        """The shared head without adapters drafts greedily; its logits are the draft's."""
        last, drafts, rows = ids.gather(1, (lengths - 1)[:, None]), [], []
        for _ in range(self.k):
            rows.append(F.linear(self.states[last], self.head))
            last = self.sampler.sample(rows[-1][:, 0], temperature=0.9, top_k=8,
                                       uniforms=torch.full((len(last),), 0.37, device="cuda"))[:, None]
            drafts.append(last)
        return torch.cat(drafts, 1), torch.cat(rows, 1)

    def target(self, ids, lengths, drafts):
        out = self.logits(torch.cat([ids.gather(1, (lengths - 1)[:, None]), drafts], 1))
        self.log.append((lengths.cpu(), drafts.cpu(), out.cpu()))
        return out


@pytest.mark.parametrize("eos", [None, 7])
def test_rollout_with_drafts_then_update(sampler, eos):
    """Rollout: a shared head with adapters gives the target's logits, the head alone the drafts, verification the tokens, all
    equal to the exact statement step by step.  Update: the adapters' log-probabilities of those tokens are the recorded ones, and a
    GRPO step's gradients reach lora_a and lora_b."""
    from rl_engine.executors.rollout import RolloutExecutor

    batch, k, new, v = 5, 3, 9, 520
    adapters = torch.tensor([0, 2, -1, 1, 2])
    model = _Policy(sampler, 64, v, 8, adapters, seed=12, k=k)
    if eos is not None:
        model.head[eos] += 0.05
    prompt = torch.tensor([[3, 1], [4, 1], [5, 9], [2, 6], [5, 3]])
    u = torch.rand(new, batch, k + 1, generator=torch.Generator().manual_seed(13))
    executor = RolloutExecutor({"temperature": 0.9, "top_k": 8})
    drafts = []

    def propose(ids, lengths):
        d = model.propose(ids, lengths)
        drafts.append(d[1].cpu())
        return d

    ids, logp, passes = executor.generate_speculative(model.target, propose, prompt.cuda(), new, u.cuda(), eos_id=eos)
    assert ids.shape == (batch, 2 + new) and logp.shape == (batch, new) and passes == len(model.log)
    rows, lps, accepted_total = [p.tolist() for p in prompt], [[] for _ in range(batch)], 0
    over = [False] * batch
    for i, (lengths, draft_ids, logits) in enumerate(model.log):
        lens = torch.tensor([0 if over[b] else min(k, new - len(lps[b]) - 1) for b in range(batch)])
        tok, acc, lp = verify_ref.verify(logits, draft_ids, u[i], drafts[i], lens, temperature=0.9, top_k=8)
        for b in range(batch):
            if over[b]:
                continue
            assert lengths[b].item() == len(rows[b])
            for j in range(int(acc[b]) + 1):
                rows[b].append(int(tok[b, j]))
                lps[b].append(float(lp[b, j]))
                accepted_total += j < int(acc[b])
                if rows[b][-1] == eos:
                    over[b] = True
                    break
            over[b] = over[b] or len(lps[b]) == new
    assert all(over) and 0 < accepted_total and passes < new
    for b in range(batch):
        full = rows[b] + [eos] * (2 + new - len(rows[b]))
        assert ids[b].tolist() == full
        assert logp[b].tolist() == pytest.approx(lps[b] + [0.0] * (new - len(lps[b])), abs=1e-4)

    # the update, on the tokens the rollout produced
    mask = torch.tensor([[j < len(l) for j in range(new)] for l in lps]).cuda()
    hidden = model.states[ids[:, 1:-1]]
    a, b = model.a.clone().requires_grad_(True), model.b.clone().requires_grad_(True)
    each = model.adapters[:, None].expand(batch, new).contiguous()
    logp_new = lora_linear_logp(sampler, hidden, model.head, a, b, ids[:, 2:].contiguous(), each, 1.5, chunk_tokens=16)
    # (the library's products round by the number of rows: two half steps of the largest logit, twice)
    top = max(out.abs().max().item() for _, _, out in model.log)
    assert ((logp_new.detach() - logp).abs()[mask] <= 8 * 2.0 ** -9 * top + 1e-4).all()
    adv = torch.randn(batch, generator=torch.Generator().manual_seed(14)).cuda()
    loss, _, dlogp = sampler.grpo_token_loss(logp_new.detach(), adv, logp_old=logp)
    logp_new.backward(torch.where(mask, dlogp, torch.zeros_like(dlogp)))
    flat = dict(hidden=hidden.view(-1, 64).cpu(), weight=model.head.cpu(), a=model.a.cpu(), b=model.b.cpu(), ids=each.view(-1).cpu(),
                tokens=ids[:, 2:].reshape(-1).cpu(), scaling=torch.full((3,), 1.5), grad=torch.where(mask, dlogp, 0 * dlogp).view(-1).cpu())
    _, _, _, da, db = _exact_logp(flat)
    bound = 2 * 2.0 ** -8 * 2 * top + 3 * 2.0 ** -8
    assert ((a.grad.cpu().double() - da).norm() / da.norm()).item() <= bound
    assert ((b.grad.cpu().double() - db).norm() / db.norm()).item() <= bound


def test_speculative_generation_of_a_greedy_policy(sampler):
    """top_k = 1 has one possible rollout: with drafts (good, bad, and outside the vocabulary) and without, it is the same."""
    from rl_engine.executors.rollout import RolloutExecutor

    g = torch.Generator().manual_seed(15)
    v, batch, new = 300, 6, 12
    table = (torch.randn(v, v, generator=g) * 3).bfloat16().cuda()
    prompt = torch.randint(0, v, (batch, 4), generator=g).cuda()
    executor = RolloutExecutor({"top_k": 1})
    want, want_lp = executor.generate(lambda seq: table[seq[:, -1]], prompt, new, eos_id=2)
    best = table.float().argmax(1)

    def target(ids, lengths, drafts):
        return table[torch.cat([ids.gather(1, (lengths - 1)[:, None]), drafts.clamp(0, v - 1)], 1)]

    def propose(ids, lengths):
        last, out = ids.gather(1, (lengths - 1)[:, None]).squeeze(1), []
        for j in range(4):
            last = best[last]
            out.append(last)
        out = torch.stack(out, 1)
        out[::3, 2] = 17
        out[1::3, 1] = v + 5
        return out, None

    ids, lp, passes = executor.generate_speculative(target, propose, prompt, new, eos_id=2)
    assert torch.equal(ids, want) and passes < new
    assert (lp - want_lp).abs().max().item() <= 1e-5
