"""One step of a beam search (lowbit.beam_select) and the reordering of its states (lowbit.beam_reorder) against plain
implementations in 64 bits.

Tolerances. Parents, labels and ends have to be equal: logits lie on a grid of 1/64 and the hypotheses' scores are drawn
until no two continuations that matter, of different hypotheses, are nearer than 1e-3. A score is off by the log-sum's
error (a sum of at most a few thousand terms per lane with exponentials good to 2^-21, so 1e-6 relative and absolute in the
logarithm) and three roundings of numbers below 128: 1e-6 + 3 * 2^-18 < 2e-5. Continuations are defined in FP32, score +
(logit - log-sum): where they are larger than 1024 in size (labels at the type's lowest value) two of them can be equal that
differ in 64 bits, so there the plain implementation rounds as the definition does, and a score is off by two roundings."""
from __future__ import annotations

import math

import pytest
import torch

from kea_kernels import _lib, lowbit

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _every(logits, scores, ended, end):
    """All continuations' scores, 64 bits, on the CPU: [clips, beams, vocab]."""
    x = logits.cpu().double()
    x = torch.where(x.isnan(), -math.inf, x)
    lse = torch.logsumexp(x, -1)
    s = scores.cpu().double()
    dead = ~(lse.isfinite() & s.isfinite())
    lse, add = torch.where(dead, 0.0, lse)[..., None], torch.where(dead, 0.0, s)[..., None]
    c = x - lse + add
    c = torch.where(c < -1024.0, ((x - lse).float() + add.float()).double(), c)   # in FP32, as defined
    c = torch.where(dead[..., None], -math.inf, c)
    if ended is not None:
        e = ended.cpu().bool()
        c = torch.where(e[..., None], -math.inf, c)
        c[..., end] = torch.where(e, torch.where(s.isfinite(), s, -math.inf), c[..., end])
    return c


def _plain(logits, scores, width, ended=None, end=None):
    c = _every(logits, scores, ended, end)
    clips, beams, vocab = c.shape
    best, at = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    parents, labels = at // vocab, at % vocab
    over = None
    if end is not None:
        over = labels == end
        if ended is not None:
            over |= ended.cpu().bool().gather(1, parents)
    return best, parents, labels, over


def _apart(c, width):
    """Clips whose choice does not hang on less than 1e-3."""
    clips, beams, vocab = c.shape
    best, at = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    best, at = best[:, :width + 1], at[:, :width + 1]
    gap = best[:, :-1] - best[:, 1:]
    return ~((gap < 1e-3) & (at[:, :-1] // vocab != at[:, 1:] // vocab) & best[:, 1:].isfinite()).any(1)


def _problem(clips, beams, vocab, dtype, width, seed, ended=False, spread=3.0, change=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.round(spread * torch.randn(clips, beams, vocab, generator=g) * 64) / 64).to(dtype)
    if change is not None:
        change(x)
    e = torch.rand(clips, beams, generator=g) < 0.3 if ended else None
    end = vocab // 2 if ended else None
    scores = torch.zeros(clips, beams)
    todo = torch.ones(clips, dtype=torch.bool)
    for _ in range(200):
        scores[todo] = -10.0 * torch.rand(int(todo.sum()), beams, generator=g)
        todo = ~_apart(_every(x, scores, e, end), width)
        if not bool(todo.any()):
            break
    assert not bool(todo.any())
    return x.to(DEV), scores.to(DEV), None if e is None else e.to(DEV), end


def _check(step, logits, scores, width, ended=None, end=None):
    best, parents, labels, over = _plain(logits, scores, width, ended, end)
    assert torch.equal(step.parents.cpu().long(), parents)
    assert torch.equal(step.tokens.cpu().long(), labels)
    got = step.scores.cpu().double()
    assert torch.equal(got.isfinite(), best.isfinite())
    fine = best.isfinite()
    tol = torch.where(best < -1024.0, 2.0 ** -22 * best.abs(), 2e-5)
    assert bool(((got - best).abs() <= tol)[fine].all())
    assert (step.ended is None) == (over is None)
    if over is not None:
        assert torch.equal(step.ended.cpu().bool(), over)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("clips,beams,vocab,width", [
    (1, 1, 1, 1), (2, 2, 2, 4), (3, 1, 7, 5), (1, 4, 1025, 4), (5, 3, 33, 3), (2, 8, 1025, 8), (1, 32, 100, 32), (7, 5, 257, 9),
    (1, 1, 5000, 32), (2, 16, 4099, 16), (1, 8, 70001, 8), (40, 8, 1025, 8), (300, 2, 129, 2), (1, 3, 40000, 1)])
def test_selection(clips, beams, vocab, width, dtype):
    x, s, _, _ = _problem(clips, beams, vocab, dtype, width, seed=vocab + beams)
    _check(lowbit.beam_select(x, s, width), x, s, width)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("clips,beams,vocab", [(4, 4, 65), (9, 8, 1025), (2, 5, 9001), (3, 1, 12)])
def test_ended_hypotheses(clips, beams, vocab, dtype):
    x, s, e, end = _problem(clips, beams, vocab, dtype, beams, seed=3, ended=True)
    _check(lowbit.beam_select(x, s, end=end, ended=e), x, s, beams, e, end)
    e[0] = True   # a clip whose hypotheses have all ended: each goes on as itself, the other places stay empty
    _check(lowbit.beam_select(x, s, end=end, ended=e), x, s, beams, e, end)


@pytest.mark.parametrize("vocab", [1024, 1025, 3001])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_any_offset(vocab, offset, dtype):
    """Labels in front of other columns (a joint's durations), rows that start at any address, clips far apart."""
    x, s, _, _ = _problem(3, 4, vocab, dtype, 4, seed=offset)
    store = torch.full((3, 2, 4, vocab + 5), 50.0, device=DEV, dtype=dtype)
    inside = store[:, 1, :, offset:offset + vocab]
    inside.copy_(x)
    _check(lowbit.beam_select(inside, s), x, s, 4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,width", [(40, 8), (1025, 8), (20000, 32), (20000, 5)])
def test_equal_logits_come_by_index(vocab, width, dtype):
    """Rows of one value, of two values, ascending and descending rows: equal continuations by their label."""
    def change(x):
        x[0] = 1.0
        x[1] = (torch.arange(vocab) % 2).to(x.dtype)
        x[2] = torch.arange(vocab).div(vocab).to(x.dtype)
        x[3] = -torch.arange(vocab).div(vocab).to(x.dtype)
        x[4, :, vocab // 2:] = 20.0
    x, s, _, _ = _problem(5, 3, vocab, dtype, width, seed=1, change=change)
    _check(lowbit.beam_select(x, s, width), x, s, width)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [20, 1025, 9000])
def test_masked_labels_and_absent_hypotheses(vocab, dtype):
    """-inf and NaN logits are masked, the type's lowest value counts as a number; a hypothesis with no label left, with a
    logit of +inf, or with an infinite or NaN score offers nothing; the places left over take what is not offered."""
    def change(x):
        low = torch.finfo(x.dtype).min
        x[0, :, 1::2] = -math.inf
        x[1, :, ::3] = math.nan
        x[2, 0] = -math.inf
        x[2, 1] = math.nan
        x[3, 2, vocab // 3] = math.inf
        x[4, :, 3:] = -math.inf                    # nine continuations for twelve places
        x[5, :, 2:] = low
        x[6, 1:] = -math.inf
    x, s, _, _ = _problem(8, 3, vocab, dtype, 12, seed=2, change=change)
    s[6, 0] = -math.inf                            # nothing at all is offered
    s[7, 1:] = -math.inf                           # a search's first step
    if vocab > 20:
        s[3, 0] = math.nan
        s[2, 2] = math.inf
    _check(lowbit.beam_select(x, s, 12), x, s, 12)


def test_large_logits_do_not_overflow():
    x, s, _, _ = _problem(2, 4, 500, torch.float32, 4, seed=9, change=lambda x: x.mul_(64).round_())
    x += 65536.0
    step = lowbit.beam_select(x, s)
    best, parents, labels, _ = _plain(x, s, 4)
    assert torch.equal(step.parents.cpu().long(), parents) and torch.equal(step.tokens.cpu().long(), labels)
    assert bool(((step.scores.cpu().double() - best).abs() <= 2.0 ** -7).all())   # the log-sum itself is near 2^16


def test_history_rows_and_graph():
    """Outputs written into rows of a history, selection and reordering captured once, replayed on new inputs."""
    clips, beams, vocab = 4, 5, 300
    x, s, _, _ = _problem(clips, beams, vocab, torch.float32, beams, seed=4)
    parents = torch.zeros(3, clips, beams, device=DEV, dtype=torch.int32)
    labels = torch.zeros_like(parents)
    scores = torch.empty(clips, beams, device=DEV)
    state = torch.randn(clips, beams, 20, device=DEV)
    run = lambda pdl: (lowbit.beam_select(x, s, out=lowbit.BeamStep(scores, parents[1], labels[1], None), pdl=pdl),  # noqa: E731
                       lowbit.beam_reorder([state], parents[1], pdl=pdl)[0])
    run(False)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        step, after = run(True)
    for seed in (5, 6):
        x2, s2, _, _ = _problem(clips, beams, vocab, torch.float32, beams, seed=seed)
        x.copy_(x2)
        s.copy_(s2)
        graph.replay()
        torch.cuda.synchronize()
        _check(step, x, s, beams)
        assert bool((parents[0] == 0).all()) and bool((parents[2] == 0).all())
        assert torch.equal(after, state.gather(1, parents[1].long()[..., None].expand(-1, -1, 20)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int64, torch.uint8, torch.bool])
@pytest.mark.parametrize("clips,beams,width", [(1, 4, 4), (3, 5, 2), (2, 2, 7)])
def test_reorder(clips, beams, width, dtype):
    g = torch.Generator().manual_seed(clips)
    parents = torch.randint(0, beams, (clips, width), generator=g, dtype=torch.int32).to(DEV)
    make = lambda *shape: torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=g).to(DEV, dtype)  # noqa: E731
    states = [make(clips, beams, n) for n in (1, 3, 16, 640, 1025, 5000)] + [make(clips, beams), make(clips, beams, 4, 6),
                                                                         make(clips, beams, 0)]
    row = torch.arange(clips, device=DEV)[:, None]
    for got, s in zip(lowbit.beam_reorder(states, parents), states):
        assert torch.equal(got, s[row, parents.long()])
    # layers first, a slice of a wider buffer, and more buffers than one launch takes
    layers = [make(3, clips, beams, 33), make(2, 2, clips, beams, 8).flatten(0, 1), make(3, clips, beams, 40)[..., 5:18]]
    for got, s in zip(lowbit.beam_reorder(layers, parents, batch_dim=1), layers):
        assert torch.equal(got, s[:, row, parents.long()])
    many = [make(clips, beams, 4) for _ in range(70)]
    out = [torch.empty(clips, width, 4, device=DEV, dtype=dtype) for _ in many]
    assert all(a is b for a, b in zip(lowbit.beam_reorder(many, parents, out=out), out))
    for got, s in zip(out, many):
        assert torch.equal(got, s[row, parents.long()])


def test_reorder_refuses_and_reports():
    parents = torch.tensor([[0, 3], [-1, 1]], device=DEV, dtype=torch.int32)
    state = torch.ones(2, 3, 10, device=DEV)
    word = torch.zeros(1, device=DEV, dtype=torch.int32)
    out = lowbit.beam_reorder([state], parents, error_word=word)[0]
    assert int(word) == _lib.DEVERR_INDEX
    assert torch.equal(out[..., 0].cpu(), torch.tensor([[1.0, 0.0], [0.0, 1.0]]))
    call = lowbit.beam_reorder
    for bad in (lambda: call([state], parents.long()), lambda: call([state], parents.cpu()), lambda: call([state[:1]], parents),
                lambda: call([state, state[:, :2]], parents), lambda: call([state.transpose(1, 2)], parents),
                lambda: call([state[..., ::2]], parents), lambda: call([state], parents, out=[]),
                lambda: call([state], parents, out=[torch.empty(2, 2, 9, device=DEV)]),
                lambda: call([state[:, :2]], parents, out=[state[:, :2]]), lambda: call([state.cpu()], parents),
                lambda: call([torch.ones(2, 4, 2, 3, 5, device=DEV).transpose(0, 1)], parents, batch_dim=2)):
        with pytest.raises(ValueError):
            bad()
    assert _lib.read_device_error() == 0


def test_refusals():
    x, s = torch.zeros(2, 3, 50, device=DEV), torch.zeros(2, 3, device=DEV)
    e = torch.zeros(2, 3, device=DEV, dtype=torch.bool)
    call = lowbit.beam_select
    for bad in (lambda: call(x.cpu(), s), lambda: call(x[0], s), lambda: call(x.double(), s), lambda: call(x.transpose(1, 2), s),
                lambda: call(x, s[:1]), lambda: call(x, s.half()), lambda: call(x, s.cpu()), lambda: call(x, s, 0),
                lambda: call(x, s, 33), lambda: call(x[..., :2], s, 7), lambda: call(x, s, end=50), lambda: call(x, s, end=-1),
                lambda: call(x, s, ended=e), lambda: call(x, s, end=1, ended=e[:, :2]), lambda: call(x, s, end=1, ended=e.float()),
                lambda: call(torch.zeros(1, 33, 4, device=DEV), torch.zeros(1, 33, device=DEV)),
                lambda: call(x, s, out=lowbit.BeamStep(s, s, s, None))):
        with pytest.raises(ValueError):
            bad()
    empty = call(x[:0], s[:0], end=3)
    assert empty.scores.shape == (0, 3) and empty.ended.shape == (0, 3)
