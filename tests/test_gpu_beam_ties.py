"""Continuations of distinct logits whose float32 scores are equal: the lower k V + v comes first, in both
forms of the selection.

A score's float32 error is far below half its step where |score| is large, so a row's few distinct logits
are chosen (a bulk value that shifts ln sum or the maximum) for scores that lie well inside a step; then a score rounded
from 64 bits is the kernel's, and the expected order is a stable sort of those."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _scores(x, score):
    """float32 scores (rounded from 64 bits) of a row's entries, None where one lies near a step's end."""
    x = x.double()
    c = score + ((x - x.max()) - (x - x.max()).exp().sum().log())
    r = c.float()
    step = torch.nextafter(r, torch.full_like(r, math.inf)).double() - r.double()
    return r if bool(((c - r.double()).abs() <= 0.4 * step).all()) else None


def _row(gen, V, dtype, score, top):
    """A row of V logits: three values of one score at random places, a bulk below, and `top` entries far above."""
    base, by, shift = (0.25, 2.0 ** -10, 0.0013) if dtype == torch.float32 else (1.0, 2.0 ** -7, 0.0625)
    kind = torch.randint(0, 8, (V,), generator=gen)
    for bulk in range(64):
        x = torch.where(kind < 3, base + by * kind, -2.0 - bulk * shift).to(dtype)
        if top:
            x[torch.randperm(V, generator=gen)[:top]] = 9.0 + bulk * shift
        c = _scores(x, score)
        if c is not None and len(set(c[(kind < 3) & (x < 8)].tolist())) == 1:
            return x, c
    raise AssertionError("no bulk value keeps the scores inside their steps")


CASES = [
    # B, K, V, n, entries above: one launch; pieces of 2048; of 8192 (a piece's end, many rows); ties in later
    # pieces; as many as can be kept
    (1, 1, 2048, 1, 0), (2, 4, 300, 5, 2), (1, 16, 500, 128, 3),
    (1, 1, 2049, 1, 0), (1, 1, 4096, 1, 0), (2, 1, 5000, 3, 1), (2, 3, 5001, 8, 2), (1, 5, 9000, 128, 1),
    (3, 8, 20011, 16, 5), (1, 1, 131072, 4, 0), (130, 8, 8200, 7, 1), (1, 128, 2100, 40, 0),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V,n,top", CASES)
def test_equal_scores_of_distinct_logits_keep_the_order_of_their_indices(B, K, V, n, top, dtype):
    from atomic_gdn2.generation import beam_step
    print(f"[gpu-test] beam ties B {B} K {K} V {V} n {n} above {top} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(B + K + V + n)
    score = -1e5 if dtype == torch.float32 else -2e6
    rows = [_row(gen, V, dtype, score, top) for _ in range(min(B * K, 24))]
    pick = [i % len(rows) for i in range(B * K)]
    logits = torch.stack([rows[i][0] for i in pick]).cuda()
    c = torch.stack([rows[i][1] for i in pick]).view(B, K * V)
    want, at = torch.sort(c, dim=-1, descending=True, stable=True)
    r = beam_step(logits, torch.full((B, K), score, device="cuda"), n=n)
    assert torch.equal(r.scores.cpu(), want[:, :n])
    flat = (r.rows.cpu() - torch.arange(B)[:, None] * K) * V + r.tokens.cpu()
    assert torch.equal(flat, at[:, :n])


def test_the_vocabularys_size_does_not_change_the_answer():
    from atomic_gdn2.generation import beam_step
    for V in (100, 2048, 4096, 50000):
        x = torch.full((1, V), -30.0, device="cuda")
        x[0, 0], x[0, 1] = 9.999999, 10.0
        assert beam_step(x, torch.full((1, 1), -100.0, device="cuda")).tokens.item() == 0, V
        x = torch.full((1, V), -math.inf, device="cuda")              # all others masked
        x[0, 30], x[0, 90] = 9.999999, 10.0
        assert beam_step(x, torch.full((1, 1), -100.0, device="cuda"), n=3).tokens[0].tolist() == [30, 90, 0], V


def test_scores_that_fall_below_float32_tie_with_masked_tokens():
    """Finite logits so far below the best that score + log-probability is -inf: they and masked tokens
    follow by index alone."""
    from atomic_gdn2.generation import beam_step
    for V in (1000, 5000):
        x = torch.full((1, V), -math.inf, device="cuda")
        x[0, 40:] = -3e38
        x[0, 900] = 3e38
        r = beam_step(x, torch.zeros((1, 1), device="cuda"), n=4)
        assert r.tokens[0].tolist() == [900, 0, 1, 2], V
        assert r.scores[0].tolist() == [0.0] + [-math.inf] * 3


def test_finished_and_dead_beams_among_equal_scores():
    from atomic_gdn2.generation import beam_step
    gen = torch.Generator().manual_seed(5)
    for V in (300, 5000):
        x, c = _row(gen, V, torch.float32, -1e5, 0)
        best = float(c.max())
        scores = torch.tensor([[best, -1e5, -math.inf, -1e5]])
        fin = torch.tensor([[True, False, False, False]])
        eos = V - 1
        full = torch.full((4, V), -math.inf)
        full[0, eos], full[1], full[3] = best, c, c
        want, at = torch.sort(full.view(-1), descending=True, stable=True)
        r = beam_step(x.expand(4, V).contiguous().cuda(), scores.cuda(), n=60, finished=fin.cuda(), eos_id=eos)
        assert torch.equal(r.scores[0].cpu(), want[:60])
        assert torch.equal(r.rows[0].cpu() * V + r.tokens[0].cpu(), at[:60])
