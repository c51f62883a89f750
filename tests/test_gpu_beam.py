"""GPU: beam selection and reordering against a plain restatement, and QtipLlama's batch over the 8-bit cache and with beams."""
import math

import pytest
import torch

import paged_reference as R
from qtip_b200 import ops
from qtip_b200.llama import LlamaShape, QtipLlama

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def select(logits, prev_scores, prev_tokens, eos, status=None):
    G, W = prev_scores.shape
    tokens, parents, scores = torch.full((G, W), -9, dtype=torch.int64, device=DEV), torch.full((G, W), -9, dtype=torch.int32, device=DEV), torch.zeros(G, W, device=DEV)
    ops.beam_select(tokens, parents, scores, logits, prev_scores, prev_tokens, eos, status=status)
    torch.cuda.synchronize()
    return tokens.cpu(), parents.cpu(), scores.cpu()


def check_select(logits, prev_scores, prev_tokens=None, eos=-1):
    """Tokens and parents are equal; scores are sums in 64 bits of fp32 numbers, rounded once, the logarithm itself rounded to fp32 from a sum whose terms
    have the exponential's error of 2^-22: one fp32 step of the logarithm (up to 2^-20 at 16) and half a step of the score."""
    G, W = prev_scores.shape
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    dev_tokens = None if prev_tokens is None else prev_tokens.to(DEV)
    tokens, parents, scores = select(logits.to(DEV), prev_scores.to(DEV), dev_tokens, eos, status)
    none_at_all = False
    for g in range(G):
        t, p, sc, none = R.select(logits[g * W:(g + 1) * W].cpu(), prev_scores[g], prev_tokens[g] if prev_tokens is not None else None, eos)
        none_at_all |= none
        assert tokens[g].tolist() == t and parents[g].tolist() == p, g
        for a, b in zip(scores[g].tolist(), sc):
            assert a == b or abs(a - b) <= 2.0 ** -20 + 2.0 ** -24 * abs(b), (g, a, b)
    assert int(status) == (2 if none_at_all else 0)


@pytest.mark.parametrize("G, W, V", [(1, 1, 1), (1, 1, 50257), (2, 3, 3), (3, 2, 1000), (1, 4, 32000), (5, 5, 32001), (2, 8, 128256), (70, 3, 999), (1, 16, 40000), (40, 16, 129),
                                     (300, 2, 2047), (9, 7, 8195)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_select_random(G, W, V, dtype):
    g = torch.Generator().manual_seed(G * V + W)
    logits = (2.5 * torch.randn(G * W, V, generator=g)).to(dtype)
    scores = -10 * torch.rand(G, W, generator=g)
    tokens = torch.randint(0, max(V, 2), (G, W), generator=g)
    check_select(logits, scores, tokens, eos=1 if V > 2 else -1)


def test_select_strides_and_in_place():
    """Rows inside a wider buffer, not aligned; the same buffers for what was and what is."""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(8, 1003, generator=g)
    scores, tokens = -5 * torch.rand(2, 4, generator=g), torch.randint(3, 900, (2, 4), generator=g)
    tokens[1, 2] = 2
    check_select(wide[:, 3:1000], scores, tokens, eos=2)
    d, s, t = wide.to(DEV)[:, 3:1000], scores.to(DEV), tokens.to(DEV)
    p = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    want = select(d, scores.to(DEV), tokens.to(DEV), 2)
    ops.beam_select(t, p, s, d, s, t, 2)
    assert torch.equal(t.cpu(), want[0]) and torch.equal(p.cpu(), want[1]) and torch.equal(s.cpu(), want[2])


@pytest.mark.parametrize("W", [1, 4, 16])
def test_select_equal_logits(W):
    """Ties: the lower beam, then the lower token; rows that are one value, two values, rising, falling."""
    V = 5000
    rows = [torch.zeros(V), (torch.arange(V) % 2).float(), torch.arange(V).float() / 100, -torch.arange(V).float() / 100]
    logits = torch.stack([rows[i % 4] for i in range(4 * W)])
    check_select(logits, torch.zeros(4, W))
    check_select(torch.cat([-logits.abs() * 0.0, logits * 0.0]), torch.zeros(8, W))            # -0 and 0


def test_select_not_finite():
    """Infinities, NaN, rows without a finite logit, beams without a score, groups without a continuation, far logits."""
    W, V, nan, inf = 4, 3000, float("nan"), float("inf")
    g = torch.Generator().manual_seed(6)
    x = torch.randn(6 * W, V, generator=g)
    x[0, ::3] = nan
    x[1, 5:2000] = inf
    x[2] = -inf
    x[3, 7] = inf
    x[4:8] = -inf                            # group 1: nothing
    x[8] = -inf
    x[8, 2999] = -300.0                      # one, far below, in the last place
    x[9] = -inf
    x[9, 0], x[9, 2000] = -1e30, 1e30
    x[10, :2900] = -1e4
    x[11] = nan
    x[12:16] *= 1e4                          # group 3
    scores = torch.zeros(6, W)
    scores[4] = torch.tensor([0.0, -inf, nan, inf])
    scores[5] = -inf
    check_select(x, scores)


# Distances of a row's larger logits from those that a warp meets first: below, at and above what 32 bits can hold of an exponential (88.7).
DISTANCES = [0, 5, 14, 20, 22, 23, 30, 40, 44, 45, 60, 70, 75, 78, 80, 81, 82, 82.5, 83, 83.5, 84, 84.5, 85, 85.3, 86, 87, 87.5, 88, 88.5, 89, 95, 120]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("low", ["first", "rising", "two values"])
def test_select_distances(dtype, low):
    """Logits that begin far below the rest of a slice, or rise through it in several batches: sums of exponentials neither overflow nor lose what counts.
    A warp's slice is 4000 logits (or 2, 4, 8 times as many); one live beam in each group, so that a lost row shows as missing continuations."""
    W, V, G = 16, 32000, len(DISTANCES)
    at = torch.arange(V) % 4000
    share = {"first": (at < 768).float(), "rising": 1 - at / 4000, "two values": (at < 768).float()}[low]
    noise = torch.zeros(G * W, V) if low == "two values" else 0.5 * torch.randn(G * W, V, generator=torch.Generator().manual_seed(11))
    logits = (noise - torch.tensor(DISTANCES).repeat_interleave(W).view(-1, 1) * share).to(dtype)
    scores = torch.full((G, W), -math.inf)
    scores[torch.arange(G), torch.arange(G) % W] = -1.0
    check_select(logits, scores)


def test_select_first_step_and_ended():
    """One live beam fills the group; ended beams stay and take one row."""
    g = torch.Generator().manual_seed(7)
    scores = torch.full((3, 5), -math.inf)
    scores[:, 0] = 0.0
    check_select(torch.randn(15, 700, generator=g), scores)
    tokens = torch.randint(3, 600, (3, 5), generator=g)
    tokens[0], tokens[1, 2] = 2, 2
    check_select(torch.randn(15, 700, generator=g), -torch.rand(3, 5, generator=g), tokens, eos=2)
    check_select(torch.randn(3, 700, generator=g), torch.zeros(3, 1), torch.full((3, 1), 2), eos=2)


def test_select_fewer_tokens_than_beams():
    scores = torch.full((2, 6), -math.inf)
    scores[:, 0] = -1.0
    check_select(torch.randn(12, 4, generator=torch.Generator().manual_seed(8)), scores)


def test_select_from_several_threads():
    """The C entry from four threads at once, on streams of their own, with widths and numbers of groups that take different clusters."""
    import threading

    from qtip_b200 import _lib
    lib, cases = _lib.load(), []
    for W, G, V in ((1, 1, 4001), (4, 3, 2000), (16, 1, 9000), (8, 40, 700)):
        logits, scores = torch.randn(G * W, V, generator=torch.Generator().manual_seed(W)).to(DEV), torch.zeros(G, W, device=DEV)
        want = select(logits, scores, None, -1)
        out = [torch.zeros(G, W, dtype=torch.int64, device=DEV), torch.zeros(G, W, dtype=torch.int32, device=DEV), torch.zeros(G, W, device=DEV)]
        cases.append((W, G, V, logits, scores, want, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    codes = []

    def run(W, G, V, logits, scores, want, out, stream):
        for _ in range(50):
            codes.append(lib.qtip_beam_select(*(t.data_ptr() for t in out), logits.data_ptr(), _lib.F32, V, scores.data_ptr(), None, G, W, V, -1, None,
                                              stream.cuda_stream))
    threads = [threading.Thread(target=run, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [0] * 200
    for c in cases:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(c[6], c[5]))


def test_select_refusals():
    G, W, V = 2, 4, 50
    z = lambda dt: torch.zeros(G, W, dtype=dt, device=DEV)  # noqa: E731
    ok = [z(torch.int64), z(torch.int32), z(torch.float32), torch.zeros(G * W, V, device=DEV), z(torch.float32), z(torch.int64), 2]
    ops.beam_select(*ok)
    for i, v, match in ((3, ok[3].double(), "unsupported dtype"), (3, ok[3][:7], "logits"), (3, torch.zeros(G * W, 2 * V, device=DEV)[:, ::2], "contiguous"), (0, z(torch.int32), "Long expected"),
                        (1, z(torch.int64), "Int expected"), (4, z(torch.float32)[:1], "shape"), (5, None, "bad argument"), (3, ok[3].cpu(), "CUDA tensors only"),
                        (3, ok[3][:1].expand(G * W, V), "shape")):
        with pytest.raises(RuntimeError, match=match):
            ops.beam_select(*(ok[:i] + [v] + ok[i + 1:]))
    z17 = lambda dt: torch.zeros(1, 17, dtype=dt, device=DEV)  # noqa: E731
    with pytest.raises(RuntimeError, match="shape"):
        ops.beam_select(z17(torch.int64), z17(torch.int32), z17(torch.float32), torch.zeros(17, V, device=DEV), z17(torch.float32))


# ------------------------------------------------------------------------------------------------------------- reordering
def reordered(t, parents, lengths, per_row, mod):
    out = t.clone()
    G, W = parents.shape
    for row in range(G * W):
        p = row // W * W + int(parents[row // W, row % W])
        n = t.shape[2]
        if lengths is not None:
            n = int(lengths[p]) % mod if mod else int(lengths[p])
            n = min(-(-n // per_row), t.shape[2])
        if p != row:
            out[row, :, :n] = t[p, :, :n]
    return out


@pytest.mark.parametrize("W", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("kind", ["survivors", "any", "permutation", "one"])
def test_reorder(W, kind):
    """Any parents, rows that change places among them; pieces that are not a multiple of 16 bytes, strided and unaligned states; lengths that end inside
    a column; rows behind them stay."""
    G = 3
    g = torch.Generator().manual_seed(W)
    parents = torch.randint(0, W, (G, W), generator=g, dtype=torch.int32)
    if kind == "survivors":
        for b in range(G):
            parents[b] = parents[b][parents[b].long()]
            keep = parents[b].unique()
            parents[b, keep.long()] = keep
    if kind == "permutation":
        parents = torch.stack([torch.randperm(W, generator=g) for _ in range(G)]).int()
    if kind == "one":
        parents[:] = W - 1
    rnd = lambda *shape: torch.randint(0, 30000, shape, generator=g).to(torch.int16)  # noqa: E731
    wide = rnd(G * W, 5, 70, 64)
    states = [(rnd(G * W, 4, 33, 40), 1, 0), (rnd(G * W, 1, 9, 2), 16, 0), (wide[:, 1:3, 3:40], 2, 32), (rnd(G * W, 1, 2100, 128), 1, 0),
              (rnd(G * W, 3, 7, 8).view(torch.int64).view(G * W, 3, 7, 2), 1, 5)]
    for lengths in (None, torch.randint(0, 2200, (G, 1), generator=g, dtype=torch.int32).expand(G, W).reshape(-1).contiguous(),
                    torch.randint(0, 40, (G * W,), generator=g, dtype=torch.int32)):
        want = [reordered(t, parents, lengths, a, m) for t, a, m in states]
        wide_dev = wide.to(DEV)
        live = [(wide_dev[:, 1:3, 3:40] if i == 2 else t.to(DEV), a, m) for i, (t, a, m) in enumerate(states)]
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.beam_reorder(live, parents.to(DEV), None if lengths is None else lengths.to(DEV), status=status)
        torch.cuda.synchronize()
        assert int(status) == 0
        for (t, _, _), w in zip(live, want):
            assert torch.equal(t.cpu(), w)
        rest = wide_dev.cpu()
        rest[:, 1:3, 3:40] = wide[:, 1:3, 3:40]
        assert torch.equal(rest, wide)


def test_reorder_parents_outside_and_refusals():
    t = torch.arange(4 * 2 * 3 * 8, dtype=torch.int32, device=DEV).view(4, 2, 3, 8)
    before, status = t.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    parents = torch.tensor([[7, -1, 0, 3]], dtype=torch.int32, device=DEV)
    ops.beam_reorder([(t, 1, 0)], parents, status=status)
    assert int(status) == 32 and torch.equal(t[[0, 1, 3]], before[[0, 1, 3]]) and torch.equal(t[2], before[0])
    ok = [(t, 1, 0)]
    for states, match in (([], "states"), (ok * 9, "states"), (ok * 2, "bad argument"), ([(t, 0, 0)], "out of range"), ([(t, 1, -1)], "out of range"), ([(t[:3], 1, 0)], "a state is"),
                          ([(t.transpose(2, 3), 1, 0)], "contiguous"), ([(t[..., :4], 1, 0)], "contiguous"), ([(t.to(torch.int8)[..., :1].contiguous(), 1, 0)], "shape"),
                          ([(t[:1].expand(4, 2, 3, 8), 1, 0)], "shape"), ([(t.cpu(), 1, 0)], "CUDA tensors only"), ([t], "tuple|state is")):
        with pytest.raises(RuntimeError, match=match):
            ops.beam_reorder(states, parents)
    now = t.clone()
    ops.beam_reorder(ok, parents.long()[:, :4].int().repeat(1, 2)[:, :4].t())        # four groups of one beam: nothing to do
    assert torch.equal(t, now)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.beam_reorder(ok, torch.zeros(2, 2, dtype=torch.int32, device=DEV).t())


def test_reorder_refuses_to_reorder_what_it_reads():
    t, L = torch.arange(4 * 6, dtype=torch.int32, device=DEV).view(4, 1, 3, 2), torch.tensor([3, 2, 1, 0], dtype=torch.int32, device=DEV)
    parents = torch.tensor([[1, 0, 3, 3]], dtype=torch.int32, device=DEV)
    before = t.clone()
    for states, p in (([(t, 1, 0), (L.view(4, 1, 1, 1), 1, 0)], parents), ([(t, 1, 0), (parents.view(4, 1, 1, 1), 1, 0)], parents)):
        with pytest.raises(RuntimeError, match="bad argument"):
            ops.beam_reorder(states, p, L)
    assert torch.equal(t, before)
    both = torch.cat([parents.view(-1), L, t.view(-1)])                   # beside one another: allowed
    live = both[8:].view(4, 1, 3, 2)
    ops.beam_reorder([(live, 1, 0)], both[:4].view(1, 4), both[4:8])
    assert torch.equal(live, reordered(before, parents, L, 1, 0)) and torch.equal(both[:8], torch.cat([parents.view(-1), L]))


# ------------------------------------------------------------------------------------------------------------ in the model
SMALL = LlamaShape(n_layers=2, hidden=512, n_heads=4, n_kv_heads=2, head_dim=128, mlp=1376, vocab=700, K=2)


def batch_logits(kv, B, steps, **kw):
    model = QtipLlama(SMALL, max_positions=64, device=DEV, seed=21)
    model.enable_batch(B, kv=kv, **kw)
    g, seen = torch.Generator().manual_seed(1), []
    model.b_pos.copy_(torch.tensor([0] * B))
    for _ in range(steps):
        model.b_token.copy_(torch.randint(0, SMALL.vocab, (B,), generator=g))
        model.step_batch()
        seen.append(model.b_logits.clone())
    model.check_status()
    return torch.stack(seen)


@pytest.mark.parametrize("kv, bound", [("int8", 0.03), ("e4m3", 0.12)])
def test_batch_over_the_8_bit_cache(kv, bound):
    """The same tokens through the batch over an fp16 cache and over the 8-bit one, up to 40 positions of blocks of 16.  A key or value is off by half of
    1/127 of the block's largest (4 deviations: 0.016 of one, spread over half a step 0.009) for int8, by 2^-4 of itself at most (0.026 spread) for e4m3;
    the logits may differ by about three times that."""
    exact, got = batch_logits(None, 3, 40), batch_logits(kv, 3, 40, block=16)
    first = (got[:15] - exact[:15]).norm() / exact[:15].norm()
    rest = (got[15:] - exact[15:]).norm() / exact[15:].norm()
    assert float(first) < 0.005          # nothing is in 8 bits yet: the angle's rounding alone
    assert float(rest) < bound


def plain_beams(model, W, prompt, steps, eos):
    """Beam search by hand: every step's logits of every beam from its whole token list, one sequence at a time."""
    beams, tokens = [(0.0, list(prompt))] + [(-math.inf, list(prompt))] * (W - 1), None
    for _ in range(steps):
        rows = []
        for _, toks in beams:
            model.reset()
            model.feed(torch.tensor(toks))
            rows.append(model.logits[0].clone())
        x = torch.stack(rows)
        last = torch.tensor([t[-1] for _, t in beams])
        toks, parents, scores, _ = R.select(x.cpu(), torch.tensor([b[0] for b in beams]), last, eos)
        beams = [(s, beams[p][1] + [t]) for t, p, s in zip(toks, parents, scores)]
    return beams


@pytest.mark.parametrize("kv", [None, "int8"])
@pytest.mark.parametrize("captured", [False, True])
def test_beams_in_the_model(kv, captured):
    """Two groups of three beams over 40 steps: the scores are those of the tokens, evaluated again by a batch without beams; the graph gives the eager
    run's tokens; sequences that share blocks read what their parents wrote."""
    W, steps, prompts = 3, 40, torch.tensor([[5, 6, 7], [300, 200, 100]])
    model = QtipLlama(SMALL, max_positions=64, device=DEV, seed=22)
    model.enable_batch(6, kv=kv, block=16)
    model.enable_beams(W, eos=-1)
    if captured:
        model.capture_batch()
    model.feed_beams(prompts)
    model.generate_batch(steps)
    model.check_status()
    tokens, scores = model.b_out_tokens[:, :3 + steps + 1].clone(), model.b_scores.clone()
    assert model.b_pos.tolist() == [3 + steps] * 6
    for row in range(6):
        assert tokens[row, :3].tolist() == prompts[row // W].tolist()
    again = QtipLlama(SMALL, max_positions=64, device=DEV, seed=22)
    again.enable_batch(6, kv=kv, block=16)
    total = torch.zeros(6, dtype=torch.float64, device=DEV)
    for i in range(3 + steps):
        again.b_token.copy_(tokens[:, i])
        again._forward_batch()
        again.b_pos.add_(1)
        if i >= 2:
            total += torch.log_softmax(again.b_logits.double(), 1).gather(1, tokens[:, i + 1:i + 2]).view(-1)
    # 41 sums of scores, each with a logarithm and a score rounded to fp32 (2^-21 and 2^-17 at 300)
    assert float((total.view(2, W) - scores.double()).abs().max()) < 41 * (2.0 ** -20 + 2.0 ** -17)
    assert len({tuple(t) for t in tokens.tolist()}) == 6


def test_beams_follow_a_search_by_hand():
    """Two beams, six steps, one sequence at a time through the batch-1 step over the fp16 cache.  (Its kernels add in another order: a seed whose
    choices are not close, scores within 2 %.)"""
    shape = SMALL
    model = QtipLlama(shape, max_positions=32, device=DEV, seed=23)
    want = plain_beams(model, 2, [11, 12], 4, -1)
    model.enable_batch(2, kv="int8", block=16)
    model.enable_beams(2)
    model.feed_beams(torch.tensor([[11, 12]]))
    model.generate_batch(3)
    got = sorted(zip(model.b_scores.view(-1).tolist(), model.b_out_tokens[:, :6].tolist()))
    for (a, t), (b, u) in zip(got, sorted((s, t) for s, t in want)):
        assert t == u and abs(a - b) < 0.02 * abs(b)


def test_beams_end():
    """Every token may end a beam: with eos as the likeliest token all beams end, keep their score and repeat it."""
    model = QtipLlama(SMALL, max_positions=32, device=DEV, seed=24)
    model.enable_batch(4, kv="e4m3", block=16)
    model.enable_beams(4)
    model.feed_beams(torch.tensor([[1, 2]]))
    eos = int(model.b_token[0])
    model.beam_eos = eos
    ended = (model.b_token == eos).nonzero().view(-1).tolist()
    before = [float(model.b_scores.view(-1)[r]) for r in ended]
    model.generate_batch(5)
    model.check_status()
    scores, tokens = model.b_scores.view(-1).tolist(), model.b_out_tokens[:, :8].tolist()
    assert any(s == before[0] and t[2:] == [eos] * 6 for s, t in zip(scores, tokens))


def test_beams_after_a_capture_are_refused():
    """A captured step without beams would go on sampling: enable_beams() wants it released first."""
    model = QtipLlama(SMALL, max_positions=32, device=DEV, seed=26)
    model.enable_batch(2)
    model.capture_batch()
    with pytest.raises(RuntimeError, match="release_graph"):
        model.enable_beams(2)
    assert model.beam_width == 0
    model.release_graph()
    model.enable_beams(2)
    model.feed_beams(torch.tensor([[1, 2]]))
    assert bool(torch.isfinite(model.b_scores).all()) and bool((model.b_scores < 0).all())


@pytest.mark.parametrize("kv", [None, "e4m3"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_second_search_starts_anew(kv, captured):
    """feed_beams() after a finished search gives what a new model gives: tokens and scores, whatever the first search left in caches, tables and tails."""
    prompts, found = [torch.tensor([[9, 8, 7, 6]]), torch.tensor([[400, 30]])], []
    for searches in (prompts, prompts[1:]):
        model = QtipLlama(SMALL, max_positions=32, device=DEV, seed=27)
        model.enable_batch(3, kv=kv, block=16)
        model.enable_beams(3)
        if captured:
            model.capture_batch()
        for p in searches:
            model.feed_beams(p)
            model.generate_batch(21)
        model.check_status()
        assert model.b_pos.tolist() == [23] * 3
        found.append((model.b_out_tokens[:, :24].clone(), model.b_scores.clone()))
    assert torch.equal(found[0][0], found[1][0]) and torch.equal(found[0][1], found[1][1])


def test_a_prompt_that_does_not_fit_is_refused():
    """... and leaves the search as it was."""
    model = QtipLlama(SMALL, max_positions=16, device=DEV, seed=29)
    model.enable_batch(2)
    model.enable_beams(2)
    model.feed_beams(torch.tensor([[1, 2, 3]]))
    before = model.b_scores.clone()
    with pytest.raises(RuntimeError, match="holds 16"):
        model.feed_beams(torch.zeros(1, 17, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="vocabulary"):
        model.feed_beams(torch.full((1, 3), SMALL.vocab))
    assert torch.equal(model.b_scores, before) and model.b_pos.tolist() == [3, 3] and model.steps_done == 3
    with pytest.raises(RuntimeError, match="holds 16"):
        model.generate_batch(14)


@pytest.mark.parametrize("prompts", [[[5, 6, 7], [300, 7, 7]], [[7], [7]]])
@pytest.mark.parametrize("captured", [False, True])
def test_prompts_that_hold_the_end_token(prompts, captured):
    """The end token in a prompt ends nothing: the first selection is that of a search without an end, in a second search too."""
    found = []
    for eos in (-1, 7):
        model = QtipLlama(SMALL, max_positions=32, device=DEV, seed=28)
        model.enable_batch(6, kv="int8", block=16)
        model.enable_beams(3, eos=eos)
        if captured:
            model.capture_batch()
        for again in range(2):
            model.feed_beams(torch.tensor(prompts))
            found.append((model.b_token.clone(), model.b_scores.clone()))
            model.generate_batch(2 if again == 0 else 0)
        model.check_status()
    for tokens, scores in found[1:]:
        assert bool(torch.isfinite(scores).all()) and torch.equal(tokens, found[0][0]) and torch.equal(scores, found[0][1])


@pytest.mark.parametrize("kv", [None, "int8"])
def test_steps_behind_the_end_of_the_log(kv):
    """step_batch() by hand, more often than there are positions: nothing is written behind the log, its rows stay the beams' tokens, the status says so."""
    model = QtipLlama(SMALL, max_positions=16, device=DEV, seed=30)
    model.enable_batch(2, kv=kv, block=16)
    model.enable_beams(2)
    for _ in range(16):
        model.step_batch()
    model.check_status()
    rows = model.b_out_tokens.tolist()
    for _ in range(5):
        model.step_batch()
    assert all(r in rows for r in model.b_out_tokens.tolist()) and model.b_pos.tolist() == [21, 21]
    assert int(model.status) & 4
    with pytest.raises(RuntimeError, match="4 = token log full"):
        model.check_status()


def test_end_token_outside_the_vocabulary_is_refused():
    """(Rows without a continuation take it as their next token.)"""
    model = QtipLlama(SMALL, max_positions=16, device=DEV, seed=30)
    model.enable_batch(2)
    for eos in (SMALL.vocab, 1 << 40):
        with pytest.raises(RuntimeError, match="outside the vocabulary"):
            model.enable_beams(2, eos=eos)
    assert model.beam_width == 0
    model.enable_beams(2, eos=SMALL.vocab - 1)


def test_pool_smaller_than_the_sequences():
    """A pool without room: the status says so, and the batch runs on with what it has."""
    model = QtipLlama(SMALL, max_positions=64, device=DEV, seed=25)
    model.enable_batch(2, kv="int8", block=16, n_blocks=3)
    for _ in range(34):
        model.step_batch()
    with pytest.raises(RuntimeError, match="8 = no free block"):
        model.check_status()
