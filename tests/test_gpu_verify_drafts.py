"""Verification of drafted tokens against a float64 walk, decision by decision (tests/draft_cases.py)."""

import math

import pytest
import torch

from falcon_perception_amd import ops
from tests.draft_cases import check_verified, random_tree, same_answers

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Step:
    """Random logits with a few likely tokens a row, drafts among them, some requests shorter than others."""

    def __init__(self, seed, B, S, V, dtype=F32, *, reach=1, probs=None, counts=None, spread=3.0):
        gen = torch.Generator().manual_seed(seed)
        x = torch.randn(B, S, V, generator=gen) * spread
        likely = torch.randint(0, V, (B, S, 6), generator=gen)
        x.scatter_(2, likely, math.log(V) + 0.5 * spread ** 2 + torch.randn(B, S, 6, generator=gen))
        self.logits = x.to(dtype)
        self.parents = torch.full((B, S), -2, dtype=torch.int32)
        self.tokens = torch.randint(0, V, (B, S), generator=gen)
        for b in range(B):
            n = S if counts is None else counts[b % len(counts)]
            tree = random_tree(gen, n, reach)
            self.parents[b, :n] = torch.tensor(tree, dtype=torch.int32)
            for j in range(1, n):
                self.tokens[b, j] = likely[b, tree[j], j % 6]
        self.uniforms = torch.rand(B, S, generator=gen)
        self.temperatures = None
        self.probs = None
        if probs is not None:
            q = torch.softmax(self.logits.double() + 0.8 * torch.randn(B, S, V, generator=gen), 2)
            self.probs = q.to(probs)
            for b in range(B):
                for j in range(1, S):
                    if self.parents[b, j] >= 0:
                        self.tokens[b, j] = int(torch.multinomial(q[b, self.parents[b, j]], 1, generator=gen))
        self.gen = gen

    def call(self, **kw):
        kw.setdefault("temperatures", None if self.temperatures is None else self.temperatures.cuda())
        kw.setdefault("draft_probs", None if self.probs is None else self.probs.cuda())
        logits = kw.pop("logits", None)
        return ops.verify_drafts(self.logits.cuda() if logits is None else logits, self.tokens.cuda(), self.parents.cuda(), self.uniforms.cuda(), **kw)

    def check(self, got=None):
        check_verified(self.call() if got is None else got, self.logits, self.tokens, self.parents, self.uniforms, self.temperatures, self.probs)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 255, 1000, 2048, 4099, 20011])
def test_chains(V, dtype):
    Step(V, 9, 5, V, dtype, counts=[5, 1, 3, 0, 4]).check()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S,reach", [(1, 1), (2, 1), (3, 3), (16, 4), (17, 17), (33, 2), (64, 8), (64, 1), (64, 64)])
def test_trees(S, reach, dtype):
    Step(S + reach, 6, S, 1500, dtype, reach=reach).check()


@pytest.mark.parametrize("probs", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 9, 777, 9001])
def test_drafts_that_were_drawn(V, dtype, probs):
    Step(V + 1, 11, 4, V, dtype, probs=probs, counts=[4, 2, 4, 1]).check()


def test_only_the_first_child_of_drawn_drafts_counts():
    Step(5, 24, 8, 300, F32, probs=F32, reach=4).check()


@pytest.mark.parametrize("probs", [None, F32])
def test_temperatures(probs):
    step = Step(6, 16, 6, 800, BF16, probs=probs, reach=1 if probs else 3)
    nan, inf = float("nan"), float("inf")
    step.temperatures = torch.tensor([0.0, 1.0, 0.3, 2.0, -1.0, nan, 0.05, 1e-30, 1e-45, inf, 1.7, 0.9, 0.0, 0.6, 1e30, -inf])
    step.check()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_greedy_takes_the_first_of_equals(dtype):
    step = Step(7, 8, 6, 5000, dtype, reach=2)
    step.temperatures = torch.zeros(8)
    top = step.logits.float().amax(2)
    for b in range(8):
        for j in range(6):
            for i in torch.randint(0, 5000, (4,), generator=step.gen).tolist():
                step.logits[b, j, i] = top[b, j] + 1
        for j in range(1, 6):
            if step.parents[b, j] >= 0 and j % 3:
                step.tokens[b, j] = int(step.logits[b, step.parents[b, j]].float().argmax())
    got = step.call()
    step.check(got)
    assert got.accepted.max() >= 2


@pytest.mark.parametrize("probs", [None, F32])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinite_logits(dtype, probs):
    """Rows that are -inf but for a few places, or everywhere; NaN; +inf; the type's lowest value."""
    step = Step(8, 12, 3, 700, dtype, probs=probs, counts=[3, 3, 1])
    inf, nan, low = float("inf"), float("nan"), torch.finfo(dtype).min
    x = step.logits
    x[0] = -inf
    x[1, :, 5:] = -inf
    x[2, :, ::2] = nan
    x[3] = nan
    x[4, :, 77] = inf
    x[5, :, 20:40] = inf
    x[6] = low
    x[7, :, 3:] = low
    x[8, 0] = -inf
    x[8, 0, 699] = 1.0
    x[9, :, 699] = inf
    x[9, :, 0] = nan
    x[10, 1:] = -inf
    step.check()
    step.temperatures = torch.zeros(12)
    step.check()
    step.temperatures = torch.full((12,), inf)
    step.check()


def test_the_same_draft_twice():
    """A token that two siblings name is refused once; drafts outside the vocabulary never stand."""
    step = Step(9, 40, 6, 50, F32, reach=6)
    step.parents[:] = torch.tensor([-1, 0, 0, 0, 0, 0])
    step.tokens[:, 2] = step.tokens[:, 1]
    step.tokens[:, 4] = step.tokens[:, 1]
    step.tokens[::3, 3] = -1
    step.tokens[1::3, 3] = 50
    step.tokens[2::3, 3] = 1 << 40
    step.uniforms[:, 1] = 0.999
    step.check()


def test_every_token_refused():
    step = Step(10, 2, 4, 3, F32)
    step.parents[:] = torch.tensor([-1, 0, 0, 0])
    step.tokens[:] = torch.tensor([0, 0, 1, 2])
    step.logits[:, 0] = torch.tensor([0.0, -float("inf"), -float("inf")])
    # of one token with all the weight every draft of it stands, whatever the number
    step.uniforms[:] = 0.9999999
    got = step.call()
    assert got.accepted.tolist() == [1, 1] and got.path[:, 1].tolist() == [1, 1]
    # three drafts that name all there is: the last one stands always
    step.logits[:, 0] = 0.0
    step.check()
    step.uniforms[:, 1:] = 2.0  # outside what is promised: nothing stands, nothing is left
    got = step.call()
    assert got.accepted.tolist() == [0, 0] and (got.tokens == -1).all() and (got.logprobs == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_numbers_at_their_ends(dtype):
    """u = 0 draws the first token that weighs something, the largest u below 1 one of the last, 1 and beyond the last."""
    V = 6001
    step = Step(11, 4, 1, V, dtype, spread=0.0)
    step.logits[:] = 0.0
    step.logits[:, :, :13] = -float("inf")
    step.logits[:, :, -4:] = -float("inf")
    step.uniforms[:, 0] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, float("nan")])
    got = step.call()
    assert got.tokens[:, 0].tolist() == [13, V - 5, V - 5, V - 5]
    assert got.accepted.tolist() == [0] * 4 and got.path[:, 0].tolist() == [0] * 4


def test_next_to_the_border():
    """Of V equal logits the token is floor(u V), wherever the sums are cut; a draft stands up to its probability and no further."""
    V = 1 << 14
    n = 512
    step = Step(12, n, 2, V, BF16, spread=0.0)
    step.logits[:] = 1.5
    i = torch.arange(n) * 31
    step.uniforms[:, 0] = i / V  # exact: the cumulative weight of tokens 0 .. i - 1
    step.tokens[:, 1] = V + 5
    got = step.call()
    assert torch.equal(got.tokens[:, 0].cpu(), i)
    step.uniforms[:, 0] = torch.nextafter(step.uniforms[:, 0], torch.tensor(0.0)).clamp(min=0.0)
    got = step.call()
    assert torch.equal(got.tokens[1:, 0].cpu(), i[1:] - 1)
    step.tokens[:, 1] = i
    step.uniforms[:, 1] = 1.0 / V
    assert got.accepted.max() == 0 and step.call().accepted.max() == 0
    step.uniforms[:, 1] = torch.nextafter(step.uniforms[:, 1], torch.tensor(0.0))
    assert step.call().accepted.min() == 1


def test_equal_distributions_always_stand():
    """p = q: every draft stands, for any number below 1 (q is exact here: of 64 equal tokens)."""
    step = Step(13, 50, 4, 64, F32, probs=F32, spread=0.0)
    step.logits[:] = 0.25
    step.probs[:] = 1.0 / 64
    step.uniforms[:, 1:] = 1.0 - 2.0 ** -24
    assert step.call().accepted.min() == 3
    step.probs[:] = 1.0  # not a distribution: drafts stand with u < 1 / 64, and where one is refused nothing is left but p itself
    step.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [600, 5003, 40000])
def test_distributions_that_differ_by_roundings(V, dtype):
    """q is p rounded to 32 bits but for two tokens, the draft among them: what is left is mostly a token's and a little everybody's, and on
    which side of 0 that little lies hangs on the last bits of Z."""
    B = 24
    step = Step(23, B, 2, V, dtype, probs=F32)
    p = torch.softmax(step.logits.double(), 2)
    q = p.clone()
    for b in range(B):
        much, less = p[b, 0].topk(2).indices.tolist()
        if b % 3:  # of every third one the little is all there is
            q[b, 0, much] += 0.5 * q[b, 0, less]
            q[b, 0, less] *= 0.5
        step.tokens[b, 1] = much
        step.uniforms[b, 1] = 1.0 - 2.0 ** -24 if b % 2 else step.uniforms[b, 1]
    step.probs = q.float()
    for b in range(0, B, 3):
        step.probs[b, 0, step.tokens[b, 1]] *= 4
    got = step.call()
    step.check(got)
    assert got.accepted.min() == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_alignments_and_strides(dtype):
    """Rows that begin at any element, lie apart, or are broadcast; probabilities alike."""
    B, S, V = 5, 4, 1537
    step = Step(14, B, S, V, dtype, probs=dtype, counts=[4, 3])
    want = step.call()
    step.check(want)
    for offset in range(0, 9):
        wide = torch.full((B, S, V + 40), float("nan"), dtype=dtype, device="cuda")
        view = wide.view(-1)[offset:offset + B * S * (V + 20)].view(B, S, V + 20)[:, :, :V]
        view.copy_(step.logits)
        q = torch.full((B, S + 1, V + 11), float("nan"), dtype=dtype, device="cuda")
        q[:, 1:, offset:offset + V] = step.probs.cuda()
        same_answers(want, step.call(logits=view, draft_probs=q[:, 1:, offset:offset + V]), V)
    same_answers(want, step.call(logits=step.logits.cuda().transpose(1, 2).contiguous().transpose(1, 2)), V)
    one = Step(15, 1, 1, V, dtype)
    rows = one.logits.cuda().expand(300, 1, V)
    u = torch.rand(300, 1)
    got = ops.verify_drafts(rows, torch.zeros(300, 1, dtype=torch.int64).cuda(), torch.full((300, 1), -1, dtype=torch.int32).cuda(), u.cuda())
    check_verified(got, one.logits.expand(300, 1, V), torch.zeros(300, 1), torch.full((300, 1), -1), u)


def test_the_answer_does_not_depend_on_the_batch():
    """One request alone, in a batch of many, and with rows cut otherwise: the same decisions."""
    step = Step(16, 64, 5, 30000, BF16, counts=[5, 4, 2])
    all_of = step.call()
    step.check(all_of)
    for b in (0, 17, 63):
        alone = ops.verify_drafts(step.logits[b:b + 1].cuda(), step.tokens[b:b + 1].cuda(), step.parents[b:b + 1].cuda(), step.uniforms[b:b + 1].cuda())
        same_answers([t[b:b + 1] for t in all_of], alone, 30000)


def test_draws_have_the_targets_distribution():
    """Chains drawn from q, verified against p: the first token of the answer is distributed as p (chi squared, 40 cells, n = 40000)."""
    V, n = 40, 40000
    gen = torch.Generator().manual_seed(17)
    p_logits, q_logits = torch.randn(V, generator=gen), torch.randn(V, generator=gen)
    p, q = torch.softmax(p_logits.double(), 0), torch.softmax(q_logits.double(), 0)
    tokens = torch.stack([torch.zeros(n, dtype=torch.int64), torch.multinomial(q, n, replacement=True, generator=gen)], 1)
    parents = torch.tensor([[-1, 0]], dtype=torch.int32).expand(n, 2).contiguous()
    u = torch.rand(n, 2, generator=gen)
    for probs in (q.float().expand(n, 2, V), None):
        got = ops.verify_drafts(p_logits.expand(n, 2, V).cuda(), tokens.cuda(), parents.cuda(), u.cuda(), draft_probs=None if probs is None else probs.cuda())
        seen = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double()
        chi = ((seen - n * p) ** 2 / (n * p)).sum().item()
        assert chi < 39 + 6 * math.sqrt(2 * 39), chi  # mean 39, variance 78


@pytest.mark.parametrize("V", [65536, 150001])
def test_large_vocabularies(V):
    Step(18, 3, 3, V, BF16).check()
    Step(19, 3, 3, V, F32, probs=F32).check()


@pytest.mark.parametrize("dtype,probs", [(F32, F32), (BF16, F16), (F16, None)])
def test_vocabularies_of_more_pieces_than_are_held(dtype, probs):
    step = Step(22, 4, 3, 1100003, dtype, probs=probs, reach=1 if probs else 3)
    step.uniforms[:, 0] = torch.tensor([0.01, 0.4, 0.95, 0.9999])
    step.check()
    step.uniforms[:, 1:] = 0.99999  # hardly any draft stands
    step.check()


def test_the_largest_vocabulary():
    step = Step(23, 1, 1, 1 << 24, F32)
    step.check()


@pytest.mark.parametrize("probs", [F32, None])
@pytest.mark.parametrize("heat", [1.0, 0.7, 30.0])
def test_far_logits(heat, probs):
    """Rows far from 0, rows that rise and fall by more than an exponential holds, NaN in front."""
    V = 9001
    step = Step(24, 9, 3, V, F32, probs=probs)
    x = step.logits
    for b, far in enumerate((-1e4, 1e4, -1e6, 1e6, 1e30)):
        x[b] += far
    ramp = torch.arange(V, dtype=torch.float32)
    x[5] += ramp
    x[6] -= 0.5 * ramp
    x[7] += 40.0 * (ramp % 2048 // 8)
    x[8, :, :6000] = float("nan")
    step.temperatures = torch.full((9,), heat)
    step.check()


def test_many_requests():
    step = Step(20, 1300, 3, 513, F32, counts=[3, 2, 0, 1])
    step.check()


def test_workspace_of_the_caller_and_no_requests():
    step = Step(21, 8, 5, 3001, F32, reach=3)
    want = step.call()
    workspace = torch.full((ops.verify_workspace_bytes(8, 5, 3001),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        for w, g in zip(want, step.call(workspace=workspace)):
            assert torch.equal(w, g)
    with pytest.raises(RuntimeError, match="workspace of [0-9]+ bytes, 16-byte aligned, is needed"):
        step.call(workspace=workspace[:-1])
    with pytest.raises(RuntimeError, match="workspace must be"):
        step.call(workspace=workspace.view(torch.int8))
    none = ops.verify_drafts(step.logits[:0].cuda(), step.tokens[:0].cuda(), step.parents[:0].cuda(), step.uniforms[:0].cuda())
    assert none.accepted.shape == (0,) and none.tokens.shape == (0, 5)


def test_refusals():
    step = Step(22, 2, 3, 40, F32)
    x, t, p, u = step.logits.cuda(), step.tokens.cuda(), step.parents.cuda(), step.uniforms.cuda()
    for args, text in [((x[:, :2], t, p, u), "logits must be"), ((x[0], t, p, u), "logits must be"), ((x[:, :, :0], t, p, u), "logits must be"),
                       ((x.double(), t, p, u), "unsupported"), ((x, t.int(), p, u), "tokens must be int64"), ((x, t[:, :2], p, u), "tokens must be"),
                       ((x, t, p.long(), u), "parents must be int32"), ((x, t, p, u.double()), "uniforms must be float32"),
                       ((x, t, p, u[:1]), "uniforms must be")]:
        with pytest.raises(RuntimeError, match=text):
            ops.verify_drafts(*args)
    with pytest.raises(RuntimeError, match="temperatures must be"):
        ops.verify_drafts(x, t, p, u, temperatures=u[0])
    with pytest.raises(RuntimeError, match="draft_probs must be"):
        ops.verify_drafts(x, t, p, u, draft_probs=x[:, :2])
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.verify_drafts(x, t, p, u, draft_probs=x.double())
