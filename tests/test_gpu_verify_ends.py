"""Verification of drafted tokens where a draw has nothing left to pass, where a greedy request's drafts were drawn, where a tree has
rows that nothing reaches, and what the drawn token's logarithm may depend on."""

import math

import pytest
import torch

from falcon_perception_amd import _native as N
from falcon_perception_amd import ops
from tests.draft_cases import check_verified
from tests.test_gpu_verify_drafts import BF16, F16, F32, Step

pytestmark = pytest.mark.gpu


def call_into(step, fill, answer=-77):
    """`verify_drafts` by the C entry point: every result and the workspace hold something before the call."""
    B, S, V = step.logits.shape
    dev = lambda t: t.cuda().contiguous()
    logits, tokens, parents, u = dev(step.logits), dev(step.tokens), dev(step.parents), dev(step.uniforms)
    probs = None if step.probs is None else dev(step.probs)
    heat = None if step.temperatures is None else dev(step.temperatures)
    made = ops.VerifiedDrafts(torch.full((B,), answer, dtype=torch.int32, device="cuda"), torch.full((B, S), answer, dtype=torch.int32, device="cuda"),
                              torch.full((B, S), answer, dtype=torch.int64, device="cuda"), torch.full((B, S), float(answer), device="cuda"))
    ws = torch.full((ops.verify_workspace_bytes(B, S, V),), fill, dtype=torch.uint8, device="cuda")
    rc = N.lib().fp_verify_drafts(
        logits.data_ptr(), logits.stride(0), logits.stride(1), N.dtype_code(logits.dtype), tokens.data_ptr(), parents.data_ptr(), u.data_ptr(),
        None if heat is None else heat.data_ptr(), None if probs is None else probs.data_ptr(), *((0, 0) if probs is None else probs.stride()[:2]),
        0 if probs is None else N.dtype_code(probs.dtype), *(t.data_ptr() for t in made), ws.data_ptr(), ws.numel(), B, S, V, N.stream_ptr(logits.device))
    N.check(rc, "fp_verify_drafts")
    torch.cuda.synchronize()
    return made, ws


@pytest.mark.parametrize("u", [1.0, 3.0, float("nan")])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("probs", [False, True])
def test_numbers_past_the_last_token(probs, dtype, u):
    """From 1 on the last token that weighs something answers, whatever the sums round to: unequal weights, and pieces behind them that
    weigh nothing."""
    B, V, some = 256, 32768, 24000
    step = Step(41, B, 2, V, dtype, probs=F32 if probs else None, spread=1.0)
    step.logits[:, :, some:] = -float("inf")
    step.logits[:, :, some - 1] = step.logits[:, :, :some].float().amax(2)
    step.parents[:] = torch.tensor([-1, 0])
    step.uniforms[:, 0] = u
    step.uniforms[:, 1] = 1e9  # the draft is refused
    step.tokens[:, 1] = 7
    if probs:
        step.probs[:, :, some - 1] = 0.0
    got, _ = call_into(step, 255)
    assert (got.accepted == 0).all()
    assert (got.tokens[:, 0] == some - 1).all()
    x = step.logits[:, 0, :].double()
    want = x[:, some - 1] - torch.logsumexp(x, 1)
    assert (got.logprobs[:, 0].cpu().double() - want).abs().max() <= 1e-5


def test_of_drawn_drafts_the_first_child_alone_decides_for_greedy_requests_too():
    step = Step(42, 12, 6, 400, F32, probs=F32, reach=6)
    step.temperatures = torch.zeros(12)
    step.parents[:] = torch.tensor([-1, 0, 0, 1, 1, 2])
    best = step.logits.argmax(2)
    step.tokens[:, 1] = (best[:, 0] + 1) % 400
    step.tokens[:, 2] = best[:, 0]
    step.tokens[::2, 1] = best[::2, 0]
    step.tokens[:, 3] = (best[:, 1] + 1) % 400
    step.tokens[:, 4] = best[:, 1]
    got = step.call()
    assert got.accepted.tolist() == [1, 0] * 6
    step.check(got)


@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_that_nothing_reaches_are_not_read(dtype, greedy):
    """Rows behind a hole, behind a second first token, and those of a sequence without a step: the workspace is left as it is for rows that name
    no parent at all."""
    step = Step(43, 4, 8, 3001, dtype)
    reached = torch.tensor([[-1, -2, 0, -2, 2, -2, -2, -2], [-1, 0, 1, -2, -2, -2, -2, -2], [-2] * 8, [-1] + [-2] * 7], dtype=torch.int32)
    others = torch.tensor([[-1, -2, 0, 1, 2, 3, -1, 6], [-1, 0, 1, -1, 3, 9, 5, 6], [-2, 0, 1, 2, 0, 0, -1, 6], [-1, 4, 1, 1, -1, 4, 5, 5]], dtype=torch.int32)
    step.temperatures = torch.zeros(4) if greedy else None
    results = []
    for parents in (reached, others):
        step.parents[:] = parents
        results.append(call_into(step, 173))
    (want, want_ws), (got, got_ws) = results
    for w, g in zip(want, got):
        assert torch.equal(w, g)
    assert torch.equal(want_ws, got_ws)
    step.check(got)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("probs", [False, True])
def test_the_drawn_tokens_logarithm_is_of_64_bit_sums(probs, dtype):
    """It is the same in every batch, bit for bit, and off by its own rounding: a token with half of the weight, 65536 others."""
    B, V = 24, 65536
    step = Step(44, B, 3, V, dtype, probs=F32 if probs else None, spread=1.0, counts=[3, 1, 2])
    gen = torch.Generator().manual_seed(45)
    x = torch.randn(B, 3, V, generator=gen)
    x[:, :, 1234] = math.log(V) + 0.5
    step.logits = x.to(dtype)
    step.uniforms[:, 1:] = 1e9  # no draft stands; of three rows both name the same token
    step.tokens[:, 1], step.tokens[:, 2] = 99, 99
    step.parents[:, 2] = torch.where(step.parents[:, 2] >= 0, 0, -2)
    if probs:
        step.probs[:, :, 1234] = 0.0
    got = step.call()
    log_p = torch.log_softmax(step.logits[:, 0].double(), 1)
    want = log_p.gather(1, got.tokens[:, :1].cpu())[:, 0]
    off = (got.logprobs[:, 0].cpu().double() - want).abs()
    # rounded once to 32 bits; weights to 2^-50 and sums over V terms
    assert (off <= want.abs() * 2.0 ** -24 + V * 2.0 ** -49).all(), off.max()
    assert (got.tokens[:, 0] == 1234).sum() >= 3
    for b0, b1 in ((0, 1), (5, 6), (7, 10), (0, B)):
        part = [step.logits[b0:b1].cuda(), step.tokens[b0:b1].cuda(), step.parents[b0:b1].cuda(), step.uniforms[b0:b1].cuda()]
        alone = ops.verify_drafts(*part, draft_probs=None if not probs else step.probs[b0:b1].cuda())
        assert torch.equal(alone.tokens, got.tokens[b0:b1]) and torch.equal(alone.logprobs, got.logprobs[b0:b1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_workspace_of_the_largest_call_serves_all(dtype):
    """Requests that end leave smaller calls behind, which are cut finer: one workspace, its bytes behind what was asked for untouched."""
    S, V = 16, 32000
    step = Step(46, 24, S, V, dtype, reach=3)
    need = ops.verify_workspace_bytes(24, S, V)
    whole = torch.full((need + 4096,), 91, dtype=torch.uint8, device="cuda")
    for B, rows in ((24, S), (6, S), (5, S), (1, S), (3, 7), (1, 1), (23, 2)):
        part = [t[:B, :rows].contiguous().cuda() for t in (step.logits, step.tokens, step.parents, step.uniforms)]
        got = ops.verify_drafts(*part, workspace=whole[:need])
        check_verified(got, *(t.cpu() for t in part))
        assert (whole[need:] == 91).all()
