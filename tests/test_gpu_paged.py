"""GPU: the key/value cache in 8-bit blocks - tables and runs, append, attention - against a plain restatement on the CPU (paged_reference)."""
import math

import pytest
import torch

import paged_reference as R
from qtip_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(*ts):
    return [t.to(DEV) for t in ts]


def run_plan(tables, lengths, new, n_blocks, block, n_tokens, extra=3):
    S = tables.shape[0]
    runs = torch.full((ops.kv_runs_capacity(n_tokens, S, block) + extra, 8), 77, dtype=torch.int32, device=DEV)
    n_runs, out, status = (torch.full((k,), 9, dtype=torch.int32, device=DEV) for k in (1, S, 1))
    status.zero_()
    t, L, n = dev(tables, lengths, new)
    ops.kv_plan(t, L, n, out, runs, n_runs, n_blocks, block, n_tokens, status=status)
    torch.cuda.synchronize()
    return t, out, runs, n_runs, status


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


PLANS = {
    "one token": (16, i32(0), i32(1), 4, 1, 2),
    "fills a block": (16, i32(15), i32(1), 4, 1, 2),
    "two blocks and a rest, from inside a block": (16, i32(5), i32(40), 9, 40, 5),
    "ends at a border": (32, i32(31, 32, 33), i32(1, 32, 31), 9, 64, 4),
    "none": (16, i32(0, 7, 16), i32(0, 0, 0), 8, 0, 3),
    "idle ones between": (64, i32(0, 200, 0, 64, 1000), i32(70, 0, 3, 64, 25), 40, 162, 17),
    "pool exhausted for the second, not for the third": (16, i32(20, 14, 3), i32(12, 2, 5), 3, 19, 3),
    "pool exhausted": (16, i32(40, 14), i32(0, 2), 2, 2, 3),
    "beyond its table": (16, i32(30, 47), i32(20, 17), 16, 37, 3),
    "up to the last token of its table": (16, i32(30, 47), i32(17, 16), 16, 33, 3),
    "negative": (16, i32(-1, 5, 18), i32(4, -2, 30), 16, 34, 4),
    "rows missing": (16, i32(0, 0), i32(20, 20), 16, 39, 4),
}


@pytest.mark.parametrize("name", PLANS)
def test_plan_cases(name):
    block, lengths, new, n_blocks, n_tokens, mb = PLANS[name]
    g = torch.Generator().manual_seed(3)
    tables = torch.full((len(lengths), mb), -1, dtype=torch.int32)
    ids, at = torch.randperm(n_blocks, generator=g), 0
    for s, n in enumerate(lengths.tolist()):
        for j in range(min(max(n, 0) // block, mb)):
            tables[s, j] = ids[at]
            at = (at + 1) % n_blocks
    check_plan(tables, lengths, new, n_blocks, block, n_tokens)


def check_plan(tables, lengths, new, n_blocks, block, n_tokens):
    want_t, want_l, want_r, want_s = R.plan(tables, lengths, new, n_blocks, block, n_tokens)
    t, out, runs, n_runs, status = run_plan(tables, lengths, new, n_blocks, block, n_tokens)
    n = int(n_runs)
    assert int(status) == want_s and n == len(want_r)
    assert out.tolist() == want_l.tolist() and torch.equal(t.cpu(), want_t) and torch.equal(runs[:n].cpu(), want_r)
    assert bool((runs[n:] == 77).all())


@pytest.mark.parametrize("seqs, block, n_blocks, hi", [(1, 128, 1, 100), (7, 16, 300, 300), (513, 32, 2500, 120), (2100, 16, 40000, 60), (130, 16, 70001, 3000), (300, 16, 90000, 3000)])
def test_plan_random(seqs, block, n_blocks, hi):
    """More sequences than threads, pools that are not a multiple of 32, tables that share blocks and name none, too few blocks at the end."""
    g = torch.Generator().manual_seed(seqs)
    rnd = lambda lo, up, *shape: torch.randint(lo, up, shape, generator=g, dtype=torch.int32)  # noqa: E731
    lengths, new = rnd(0, hi, seqs), rnd(0, 40, seqs)
    lengths[::5] = 0
    mb = (hi + 40) // block + 1
    tables = rnd(0, n_blocks, seqs, mb)
    tables[seqs // 2, 0] = n_blocks          # names no block (if it is among the live ones: status 16)
    check_plan(tables, lengths, new, n_blocks, block, int(new.sum()) - (3 if seqs > 500 else 0))


def test_plan_shares_and_releases():
    tables = torch.tensor([[0, 1, -1], [0, 1, -1], [2, -1, -1]], dtype=torch.int32)
    t, out, runs, n_runs, status = run_plan(tables, i32(32, 40, 0), i32(16, 8, 16), 5, 16, 40)
    # the third has released block 2; blocks 0 and 1 are held once for two
    assert t.tolist() == [[0, 1, 2], [0, 1, 3], [4, -1, -1]] and out.tolist() == [48, 48, 16] and int(status) == 0


@pytest.mark.parametrize("lengths, new, n_blocks, served", [
    ([16, 15], [32, 1], 2, [16, 16]),                                      # needs of 2 and 1, one block free: the second is served
    ([0, 0, 0, 0], [48, 16, 32, 16], 2, [0, 16, 0, 16]),
    ([0, 31, 0, 7, 15], [15, 1, 200, 3, 1], 2, [15, 32, 0, 10, 15]),       # the second takes the one that is free, the last finds none
    ([0, 31, 0, 7, 15], [15, 17, 200, 3, 1], 2, [15, 31, 0, 10, 16]),      # those that need no block are served too
    ([0] * 1500, [16 + 16 * (i % 3) for i in range(1500)], 1004, None),
    ([0] * 1200, [16] * 1023 + [48] + [16] * 176, 1025, None),             # across the 1024 sequences that are planned at a time
    ([0] * 1200, [16] * 1000 + [48] * 24 + [32] * 176, 1001, None),
    ([0] * 1200, [16] * 1000 + [48] * 24 + [32] * 100 + [16] * 76, 1001, None),
])
def test_plan_refused_sequences_take_nothing(lengths, new, n_blocks, served):
    """Where the pool is exhausted, a sequence that does not fit is left out and takes no block from the ones behind it."""
    block, S = 16, len(lengths)
    tables = torch.full((S, 16), -1, dtype=torch.int32)
    held = 0
    for s, n in enumerate(lengths):
        for j in range(n // block):
            tables[s, j] = held
            held += 1
    free, want, out, names = n_blocks - held, 0, [], tables.clone()
    for s in range(S):
        need = (lengths[s] + new[s]) // block - lengths[s] // block
        if want + need > free and need:
            out.append(lengths[s])
            continue
        for j in range(need):
            names[s, lengths[s] // block + j] = held + want + j
        want += need
        out.append(lengths[s] + new[s])
    assert served is None or out == served
    t, after, runs, n_runs, status = run_plan(tables, i32(*lengths), i32(*new), n_blocks, block, sum(new))
    assert after.tolist() == out and torch.equal(t.cpu(), names) and int(status) == 8
    first_row = [sum(new[:s]) for s in range(S)] if S < 10 else torch.tensor(new).cumsum(0).sub(torch.tensor(new)).tolist()
    rows = runs[:int(n_runs)].tolist()
    assert [r[0] for r in rows] == sorted(r[0] for r in rows) and sum(r[3] for r in rows) == sum(o - n for o, n in zip(out, lengths))
    for seq, row, pos, count, b, _, _, _ in rows:
        assert row == first_row[seq] + pos - lengths[seq] and out[seq] >= pos + count
        assert b == (names[seq, pos // block] if (pos + count) % block == 0 else b) and ((pos + count) % block == 0 or b < 0)


def test_plan_refusals():
    t, L = torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    out, runs, n = torch.zeros_like(L), torch.zeros(10, 8, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ok = [t, L, torch.ones_like(L), out, runs, n, 8, 16, 2]
    ops.kv_plan(*ok)

    def bad(i, v, match):
        with pytest.raises(RuntimeError, match=match):
            ops.kv_plan(*(ok[:i] + [v] + ok[i + 1:]))
    bad(3, L, "bad argument")                       # in place
    bad(7, 24, "shape")
    bad(6, 0, "shape")
    bad(6, 1600001, "shape")
    bad(8, 200, "workspace")                        # too few rows of runs
    bad(8, -1, "shape")
    bad(0, t.long(), "Int expected")
    bad(0, t.t(), "contiguous")
    bad(1, L[:1], "shape")
    bad(4, runs[:, :7], "shape")
    bad(1, L.cpu(), "CUDA tensors only")


# ---------------------------------------------------------------------------------------------------------------- append
def make_inputs(T, heads, kv, hd, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(T, w * hd, generator=g).mul(f).half() for w, f in ((heads, 1.0), (kv, 2.0 * scale), (kv, scale)))
    return q, k, v


def inv_freq(hd, theta=10000.0):
    return theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)


def gpu_append(parts, tables, lengths, new, q, k, v, kind, n_blocks, block, freq, q_out=None, status=None):
    T = q.shape[0]
    t, out, runs, n_runs, _ = run_plan(tables, lengths, new, n_blocks, block, T)
    q_out = torch.empty_like(q) if q_out is None else q_out
    ops.rope_kv_append_paged(q_out, q, k, v, *parts, runs, n_runs, freq, kind, status=status)
    return t.cpu(), out.cpu(), q_out


APPENDS = [  # heads, kv, hd, block, kind, pieces of each sequence
    (4, 4, 128, 32, "int8", [[1] * 35]),
    (8, 2, 64, 16, "e4m3", [[40, 1, 7], [0, 16, 15], [3, 3, 60]]),
    (6, 2, 128, 64, "e4m3", [[63, 1, 1], [64, 64, 64], [200, 5, 123]]),
    (5, 5, 64, 128, "int8", [[127, 2, 130], [128, 0, 0], [1, 255, 1]]),
    (32, 1, 128, 16, "int8", [[5, 44, 16]]),
]


@pytest.mark.parametrize("heads, kv, hd, block, kind, pieces", APPENDS)
def test_append_bits(heads, kv, hd, block, kind, pieces):
    """Every code, scale, tail row and rotated query, for tokens that come in pieces: equal in every bit, and what is not written stays."""
    S, rounds = len(pieces), len(pieces[0])
    total = [sum(p) for p in pieces]
    mb, n_blocks = max(total) // block + 1, sum(n // block for n in total) + 2
    ref = R.Cache(S, n_blocks, kv, hd, block, kind)
    for t in (ref.data, ref.scales, ref.tail_k, ref.tail_v):
        t.copy_(torch.randint(0, 100, t.shape, generator=torch.Generator().manual_seed(1)).to(t.dtype))
    parts = ref.parts(DEV)
    freq = inv_freq(hd, 500000.0)
    tables, lengths = torch.full((S, mb), -1, dtype=torch.int32), torch.zeros(S, dtype=torch.int32)
    for r in range(rounds):
        new = i32(*[p[r] for p in pieces])
        T = int(new.sum())
        if T == 0:
            continue
        q, k, v = make_inputs(T, heads, kv, hd, 10 * r + hd)
        tables, after, q_out = gpu_append(parts, tables, lengths, new, *dev(q, k, v), kind, n_blocks, block, freq.to(DEV))
        t0 = 0
        want_q = torch.empty_like(q)
        for s in range(S):
            for i in range(int(new[s])):
                pos = int(lengths[s]) + i
                want_q[t0] = R.rotate(q[t0].view(heads, hd), pos, freq).view(-1)
                ref.append(s, pos, R.rotate(k[t0].view(kv, hd), pos, freq), v[t0].view(kv, hd), tables[s])
                t0 += 1
        lengths = after
        assert torch.equal(q_out.cpu(), want_q)
        assert torch.equal(parts[0].cpu(), ref.data) and torch.equal(parts[1].cpu(), ref.scales)
        for s in range(S):          # rows in use (behind them a tail may hold what was there)
            n = int(lengths[s]) % block
            assert torch.equal(parts[2][s, :, :n].cpu(), ref.tail_k[s, :, :n])
            a, b = (x[s].permute(0, 1, 3, 2).reshape(kv, block, hd)[:, :n] for x in (parts[3].cpu(), ref.tail_v))
            assert torch.equal(a, b)
    assert lengths.tolist() == total


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_odd_values(kind):
    """Zeros, the smallest and the largest fp16, an infinity and a NaN in one head's block; a position beyond a million; in place; strided rows."""
    kv, hd, block, S = 4, 64, 16, 1
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(16, 3 * kv * hd + 8, generator=g).half()
    qkv[:, kv * hd:kv * hd + hd] = 0                                   # head 0 of k: zeros
    qkv[:, 2 * kv * hd + hd:2 * kv * hd + 2 * hd] = 2.0 ** -24         # head 1 of v
    qkv[3, 2 * kv * hd + 2 * hd] = 65504.0
    qkv[7, kv * hd + 2 * hd + 5] = float("inf")
    qkv[9, 2 * kv * hd + 3 * hd + 1] = float("nan")
    d = qkv.to(DEV)
    q, k, v = d[:, :kv * hd], d[:, kv * hd:2 * kv * hd], d[:, 2 * kv * hd:3 * kv * hd]
    ref = R.Cache(S, 1, kv, hd, block, kind)
    parts = ref.parts(DEV)
    start = (1 << 20) + 16                                             # (the table is not long enough: the runs are made here)
    runs = torch.tensor([[0, 0, start, 16, 0, -1, 0, 0]], dtype=torch.int32, device=DEV)
    freq = inv_freq(hd)
    ops.rope_kv_append_paged(q, q, k, v, *parts, runs, torch.ones(1, dtype=torch.int32, device=DEV), freq.to(DEV), kind)
    table = {start // block: 0}
    for i in range(16):
        x = qkv[i]
        ref.append(0, start + i, R.rotate(x[kv * hd:2 * kv * hd].view(kv, hd), start + i, freq), x[2 * kv * hd:3 * kv * hd].view(kv, hd), table)
        assert torch.equal(d[i, :kv * hd].cpu(), R.rotate(x[:kv * hd].view(kv, hd), start + i, freq).view(-1))
    assert torch.equal(parts[0].cpu(), ref.data)
    assert torch.equal(parts[1].cpu().nan_to_num(-7.0), ref.scales.nan_to_num(-7.0))
    assert bool(parts[1][0, 2, 0].isnan()) and bool(parts[1][0, 3, 1].isnan()) and float(parts[1][0, 0, 0]) > 0
    assert torch.equal(d[:, kv * hd:].cpu().nan_to_num(5.0), qkv[:, kv * hd:].nan_to_num(5.0))


def test_append_runs_outside_are_skipped():
    """Runs that no plan makes: nothing is read or written for them, and the status says so."""
    kv, hd, block = 2, 64, 16
    ref = R.Cache(2, 3, kv, hd, block, "int8")
    parts = ref.parts(DEV)
    q, k, v = dev(*make_inputs(4, kv, kv, hd, 0))
    for run in ([2, 0, 0, 1, -1], [-1, 0, 0, 1, -1], [0, 4, 0, 1, -1], [0, 3, 0, 2, -1], [0, -1, 0, 1, -1], [0, 0, 15, 2, -1], [0, 0, -4, 1, -1], [0, 0, 0, 4, 1],
                [0, 0, 15, 1, 3], [0, 0, 0, 17, -1]):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        q_out = torch.full_like(q, 3.0)
        ops.rope_kv_append_paged(q_out, q, k, v, *parts, torch.tensor([run + [-1, 0, 0]], dtype=torch.int32, device=DEV),
                                 torch.ones(1, dtype=torch.int32, device=DEV), inv_freq(hd).to(DEV), "int8", status=status)
        assert int(status) == 1 and bool((q_out == 3.0).all()), run
    for a, b in zip(parts, ref.parts("cpu")):
        assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------------------------------------------------- attention
def random_cache(S, n_blocks, kv, hd, block, kind, seed, v_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    c = R.Cache(S, n_blocks, kv, hd, block, kind)
    x = torch.randn(c.data.shape, generator=g)
    c.data = (x * 36).round().clamp(-127, 127).add(128).to(torch.uint8) if kind == "int8" else (x * 128).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    c.scales = 3.5 / R.TOP[kind] * torch.exp(0.5 * torch.randn(n_blocks, kv, 4, generator=g))
    c.scales[:, :, 1] *= v_scale
    c.tail_k, c.tail_v = torch.randn(c.tail_k.shape, generator=g).half(), (v_scale * torch.randn(c.tail_v.shape, generator=g)).half()
    return c


def check_attention(c, lengths, tables, heads, seed=0, q_gain=1.5, got=None):
    """Off by the rounding to fp16 (half a step, 2^-11 of the value) and by what the weights' errors move: scores are sums of 128 products in fp32 with the
    exponential's 2^-22, weights two parts of fp16 (2^-22): below 2^-15 of the largest value, with scores of this size."""
    S = len(lengths)
    q = (q_gain * torch.randn(S, heads * c.hd, generator=torch.Generator().manual_seed(seed))).half()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full((S, heads * c.hd), 7.0, dtype=torch.float16, device=DEV)
    ops.attn_decode_paged(out, q.to(DEV), *c.parts(DEV), tables.to(DEV), i32(*lengths).to(DEV), c.kind, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    out = out.cpu().double().view(S, heads, c.hd)
    for s, n in enumerate(lengths):
        want = c.attend(q[s].view(heads, c.hd), s, n, tables[s])
        if n == 0:
            assert bool((out[s] == 0).all())
            continue
        rep = heads // c.kv
        for h in range(c.kv):
            top = float(c.values(s, n, tables[s], h, 1).abs().max())
            w, y = want[h * rep:(h + 1) * rep], out[s, h * rep:(h + 1) * rep]
            off = (y - w).abs() - (2.0 ** -11 * w.abs() + 2.0 ** -15 * top + 2.0 ** -25)
            assert float(off.max()) <= 0, (s, n, h, float(off.max()), top)


def tables_for(lengths, block, n_blocks, mb, seed=0):
    """Different places in the pool; behind the complete blocks, numbers of no block."""
    ids, at = torch.randperm(n_blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32), 0
    t = torch.full((len(lengths), mb), 1 << 30, dtype=torch.int32)
    for s, n in enumerate(lengths):
        t[s, :n // block] = ids[at:at + n // block]
        at += n // block
    return t


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 160, 255, 256, 257, 300]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads, kv", [(3, 3), (6, 2), (16, 2), (9, 1), (17, 1)])
def test_attention_edges(heads, kv, hd, block, kind):
    """Lengths around every border of blocks, tiles and pieces; 1 to 17 query heads on a key/value head."""
    mb = 300 // block
    n_blocks = sum(n // block for n in EDGES)
    c = random_cache(len(EDGES), n_blocks, kv, hd, block, kind, heads)
    check_attention(c, EDGES, tables_for(EDGES, block, n_blocks, mb), heads)


@pytest.mark.parametrize("lengths, heads, kv, hd, block, kind", [
    ([5000], 4, 1, 128, 16, "int8"), ([9000, 0, 3], 8, 2, 64, 64, "e4m3"), ([2047, 1, 6001, 512], 40, 2, 128, 32, "int8"),
    ([333] * 67, 2, 2, 64, 16, "e4m3"), ([20000], 1, 1, 128, 128, "int8"), ([0] * 9, 4, 4, 128, 32, "int8"),
])
def test_attention_split(lengths, heads, kv, hd, block, kind):
    """Sequences that several CTAs share, and CTAs that go through several sequences."""
    n_blocks = sum(n // block for n in lengths) + 1
    c = random_cache(len(lengths), n_blocks, kv, hd, block, kind, 5)
    check_attention(c, lengths, tables_for(lengths, block, n_blocks, max(lengths) // block + 1), heads)


def marked_cache(S, n_blocks, kv, hd, block, kind, seed):
    """A pool in which block j's values are one number, different from block to block, in dim j of 64 (and 64 + j), zero elsewhere: a dim of the result is the
    weight of the tokens whose blocks carry it, so a tile that is left out or counted twice shows."""
    c = random_cache(S, n_blocks, kv, hd, block, kind, seed)
    one = torch.full((block, hd), 128 if kind == "int8" else 0, dtype=torch.uint8)
    for j in range(n_blocks):
        codes = one.clone()
        codes[:, [d for d in range(hd) if d % 64 == j % 64]] = 255 if kind == "int8" else 0x7E          # the largest value
        c.data[j, :, :, 1] = R.pack(codes, 1)
        c.scales[j, :, 1] = (1 + j % 7 / 8) / R.TOP[kind]
    c.tail_v = c.tail_v.abs()
    return c


def sections(lengths, block, n_blocks, mb, tokens):
    """Tables in which consecutive stretches of `tokens` tokens name one block."""
    t = torch.full((len(lengths), mb), 1 << 30, dtype=torch.int32)
    for s, n in enumerate(lengths):
        t[s, :n // block] = ((torch.arange(n // block) * block // tokens * 5 + s) % n_blocks).int()
    return t


def check_marked(c, lengths, heads, tokens):
    """All values are at least 0, so every sum keeps its relative error: half a step of the result (2^-11); scores of below 2^4 bits, off by 2^-19 in fp32, with
    the exponential's and the two parts' 2^-22: 2^-18 in a weight; up to 2^9 additions of a lane and 2^9 of the parts at 2^-24 to 2^-23 each: 2^-13."""
    mb = max(lengths) // c.block
    tables = sections(lengths, c.block, c.data.shape[0], max(mb, 1), tokens)
    q = torch.randn(len(lengths), heads * c.hd, generator=torch.Generator().manual_seed(3)).mul(0.5).half().to(DEV)
    out, status = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device=DEV)
    parts = c.parts(DEV)
    ops.attn_decode_paged(out, q, *parts, tables.to(DEV), i32(*lengths).to(DEV), c.kind, status=status)
    assert int(status) == 0
    rep, lut = heads // c.kv, R.code_values(c.kind).to(DEV)
    for s, n in enumerate(lengths):
        got = out[s].double().view(heads, c.hd)
        if n == 0:
            assert bool((got == 0).all())
            continue
        ids = tables[s, :n // c.block].long().to(DEV)
        for h in range(c.kv):
            kv = []
            for w, tail in ((0, parts[2][s, h]), (1, parts[3][s, h].permute(0, 2, 1).reshape(c.block, c.hd))):
                pool = lut[parts[0][:, h, :, w][..., R.places(w, c.hd).to(DEV)].long()].view(-1, c.block, c.hd) * parts[1][:, h, w].double()[:, None, None]
                kv.append(torch.cat([pool[ids].reshape(-1, c.hd), tail[:n % c.block].double()]))
            p = torch.softmax(q[s].view(heads, c.hd)[h * rep:(h + 1) * rep].double() @ kv[0].T / math.sqrt(c.hd), 1)
            want = p @ kv[1]
            off = (got[h * rep:(h + 1) * rep] - want).abs() - ((2.0 ** -11 + 2.0 ** -12) * want + 2.0 ** -25)
            assert float(off.max()) <= 0, (s, n, h, float(off.max()), float(want.max()))


@pytest.mark.parametrize("heads, kv, hd, block, kind, lengths", [
    (4, 4, 128, 16, "int8", [40001, 0, 131071, 7, 90000, 1, 200016, 33333, 131072]),           # up to 8 query heads on one, 128 dims: from 71040 tiles
    (32, 2, 128, 32, "e4m3", [300033, 1000, 0, 262144, 129, 250001]),                           # 16 of them: from 47360
    (17, 1, 64, 64, "int8", [700001, 0, 450000, 64, 500063]),                                   # two groups, 64 dims: from 94720
    (4, 2, 64, 16, "e4m3", [500001, 1000, 0, 262144, 15, 850001, 31, 750016]),                  # 64 dims: from 142080
])
def test_attention_ranges_in_waves(heads, kv, hd, block, kind, lengths):
    """So many tiles that the CTAs take them in waves of smaller ranges; pairs that cross from one wave into the next; sequences of none between."""
    groups = -(-heads // kv // 16)
    tiles = sum((n // block * block + 31) // 32 + (n % block + 15) // 16 + 4 for n in lengths if n) * kv * groups
    ctas = torch.cuda.get_device_properties(0).multi_processor_count * (3 if heads // kv <= 8 else 2)
    assert tiles >= ctas * (160 if hd == 128 else 320)
    check_marked(marked_cache(len(lengths), 67, kv, hd, block, kind, 31), lengths, heads, 2000)


@pytest.mark.parametrize("heads, hd, kind", [(4, 128, "int8"), (16, 128, "e4m3"), (1, 64, "int8")])
def test_attention_joins_many_parts(heads, hd, kind):
    """A pair in more than 256 parts (a CTA's threads): the join goes through them in steps, with what it has so far carried on."""
    check_marked(marked_cache(2, 67, 1, hd, 64, kind, 32), [131071, 5], heads, 512)


@pytest.mark.parametrize("gain", [0.0, 30.0])
def test_attention_flat_and_peaked(gain):
    """All scores equal; one score far above the others (scores of some hundreds: their fp32 sums are off by 2^-14, the allowance for weights holds as
    all weight is on one token or on ones that differ by more)."""
    lengths = [700, 40]
    c = random_cache(2, 60, 2, 128, 16, "int8", 6)
    if gain == 0.0:
        check_attention(c, lengths, tables_for(lengths, 16, 60, 44), 4, q_gain=0.0)
        return
    tables = tables_for(lengths, 16, 60, 44)
    c.tail_k[:, :, 3] *= 8                               # one token of each tail far away in the direction of q
    q = torch.cat([c.tail_k[s, h, 3].repeat(2) for s in range(2) for h in range(2)]).view(2, -1)
    out = torch.zeros(2, 4 * 128, dtype=torch.float16, device=DEV)
    ops.attn_decode_paged(out, q.to(DEV), *c.parts(DEV), tables.to(DEV), i32(*lengths).to(DEV), "int8")
    for s in range(2):
        want = c.attend(q[s].view(4, 128), s, lengths[s], tables[s])
        assert torch.equal(out[s].cpu().view(4, 128), want.half())       # the token's value itself


@pytest.mark.parametrize("v_scale", [2.0 ** -12, 64.0])
def test_attention_small_and_large_values(v_scale):
    lengths = [100, 37]
    c = random_cache(2, 16, 1, 64, 16, "int8", 7, v_scale)
    check_attention(c, lengths, tables_for(lengths, 16, 16, 7), 2)


def test_attention_scales_of_many_sizes():
    """Blocks whose V scales differ by 2^20: the small ones' share is below what is allowed, the large ones' exact."""
    lengths = [200]
    c = random_cache(1, 13, 2, 128, 16, "int8", 8)
    c.scales[:, :, 1] *= 2.0 ** torch.randint(-20, 1, (13, 1)).float()
    check_attention(c, lengths, tables_for(lengths, 16, 13, 13), 2)


def test_attention_nothing_hidden_is_seen():
    """NaN in tail rows behind the last token, in blocks of other sequences and in a sequence of length 0's tail."""
    block, lengths = 32, [70, 32, 0]
    c = random_cache(3, 8, 2, 64, block, "e4m3", 9)
    tables = tables_for(lengths, block, 4, 5)
    for s, n in enumerate(lengths):
        c.tail_k[s, :, n % block:] = float("nan")
        v = c.tail_v[s].permute(0, 1, 3, 2).reshape(2, block, 64)
        v[:, n % block:] = float("nan")
        c.tail_v[s] = v.view(2, block // 2, 2, 64).permute(0, 1, 3, 2)
    c.scales[4:] = float("nan")
    check_attention(c, lengths, tables, 4)


def test_attention_not_finite():
    """A block that stands for NaN makes its sequence and head NaN, no other; a table that names no block its sequence, with the status."""
    lengths, block = [64, 64], 32
    c = random_cache(2, 4, 2, 64, block, "int8", 10)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    q = torch.randn(2, 4 * 64).half().to(DEV)
    good = torch.empty_like(q)
    ops.attn_decode_paged(good, q, *c.parts(DEV), tables.to(DEV), i32(*lengths).to(DEV), "int8")
    parts = c.parts(DEV)
    parts[1][1, 0, 1] = float("nan")
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.attn_decode_paged(out, q, *parts, tables.to(DEV), i32(*lengths).to(DEV), "int8", status=status)
    assert bool(out[0, :128].isnan().all()) and torch.equal(out[0, 128:], good[0, 128:]) and torch.equal(out[1], good[1]) and int(status) == 0
    for wrong in (-1, 4, 1 << 30):
        tables[1, 0] = wrong
        ops.attn_decode_paged(out, q, *c.parts(DEV), tables.to(DEV), i32(*lengths).to(DEV), "int8", status=status)
        assert int(status) == 16 and torch.equal(out[0], good[0]) and bool(out[1].isnan().all())
        status.zero_()
    for n in (-5, 96):                                  # no such length: as none, with the status
        ops.attn_decode_paged(out, q, *c.parts(DEV), torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), i32(64, n).to(DEV), "int8", status=status)
        assert int(status) == 1 and torch.equal(out[0], good[0]) and bool((out[1] == 0).all())
        status.zero_()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("gain", [100.0, 1e3, 1e4, 1.1e4, 1.3e4, 1.5e4, 2e4, 6e4])
def test_attention_very_large_scores(gain, kind):
    """Scores of 10^5 to 6 * 10^10 (128 products of gain * gain, / sqrt(128), in bits of the exponent): all weight on the token that looks where the
    query does, or in equal parts on two of them, in blocks and in the tail; nothing overflows.  The weights are then 1, or 1/2 each, but for the two parts
    of fp16 (2^-22) and the exponential's 2^-22; a value is off by the rounding to fp16 (2^-11 of itself, 2^-25 below 2^-14) and by 2^-20 of itself, far below the
    2^-13 allowed here."""
    kv, hd, block = 2, 128, 16
    g = torch.Generator().manual_seed(int(gain))
    places = [[3], [40, 150], [163], [5, 9], [161, 162], [0, 100]]           # of sequences of 165 tokens: ten blocks and five rows of the tail
    S, n = len(places), 165
    u = torch.where(torch.rand(kv, hd, generator=g) < 0.5, -1.0, 1.0)
    c = R.Cache(S, S * 10, kv, hd, block, kind)
    tables = torch.arange(S * 10, dtype=torch.int32).view(S, 10)
    for s in range(S):
        for t in range(n):
            k = gain * u if t in places[s] else 0.01 * gain * torch.randn(kv, hd, generator=g)
            c.append(s, t, k.half(), torch.randn(kv, hd, generator=g).half(), tables[s])
    q = (gain * u).half().repeat_interleave(2, 0).view(1, -1).expand(S, -1).contiguous()
    out, status = torch.zeros(S, 4 * hd, dtype=torch.float16, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.attn_decode_paged(out, q.to(DEV), *c.parts(DEV), tables.to(DEV), i32(*[n] * S).to(DEV), kind, status=status)
    assert int(status) == 0
    for s in range(S):
        for h in range(4):
            v = c.values(s, n, tables[s], h // 2, 1)[places[s]]
            k = c.values(s, n, tables[s], h // 2, 0)[places[s]]
            assert len(k) == 1 or torch.equal(k[0], k[1])                    # (of one size, in blocks too: the block's largest has its top code)
            off = (out[s].cpu().double().view(4, hd)[h] - v.mean(0)).abs() - ((2.0 ** -11 + 2.0 ** -13) * v.abs().amax(0) + 2.0 ** -25)
            assert float(off.max()) <= 0, (s, h, float(off.max()))


def test_attention_keys_not_finite():
    """A block whose keys stand for NaN, with finite values, makes its sequence and head NaN, no other."""
    lengths, block = [64, 64], 32
    c = random_cache(2, 4, 2, 64, block, "int8", 13)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 4 * 64).half().to(DEV)
    good, out, parts = torch.empty_like(q), torch.empty_like(q), c.parts(DEV)
    ops.attn_decode_paged(good, q, *parts, tables, i32(*lengths).to(DEV), "int8")
    parts[1][1, 0, 0] = float("nan")
    ops.attn_decode_paged(out, q, *parts, tables, i32(*lengths).to(DEV), "int8")
    assert bool(out[0, :128].isnan().all()) and torch.equal(out[0, 128:], good[0, 128:]) and torch.equal(out[1], good[1])


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_attention_values_not_finite_in_the_tail(value):
    """Their dim is not finite, the other dims and the other heads are what they would be."""
    lengths, block = [70], 32
    c = random_cache(1, 2, 2, 64, block, "int8", 14)
    tables = torch.tensor([[0, 1]], dtype=torch.int32)
    q = torch.randn(1, 4 * 64, generator=torch.Generator().manual_seed(5)).half()
    out = torch.zeros(1, 4 * 64, dtype=torch.float16, device=DEV)
    want = c.attend(q.view(4, 64), 0, 70, tables[0])
    top = float(max(c.values(0, 70, tables[0], h, 1).abs().max() for h in range(2)))
    c.tail_v[0, 1, 2, 17, 1] = value                         # token 69, key/value head 1, dim 17
    ops.attn_decode_paged(out, q.to(DEV), *c.parts(DEV), tables.to(DEV), i32(*lengths).to(DEV), "int8")
    out = out.cpu().view(4, 64).double()
    assert not bool(torch.isfinite(out[2:, 17]).any())
    out[2:, 17] = want[2:, 17]
    # as check_attention: half a step of fp16 and 2^-15 of the largest value
    assert float(((out - want).abs() - (2.0 ** -11 * want.abs() + 2.0 ** -15 * top + 2.0 ** -25)).max()) <= 0


def test_attention_strides_streams_and_graph():
    """Rows inside wider buffers, tails inside a cache of several layers; two streams at once without a workspace; a captured call replayed with other
    lengths; the same bits each time."""
    S, heads, kv, hd, block = 3, 4, 2, 128, 16
    lengths = [900, 17, 300]
    n_blocks = sum(n // block for n in lengths)
    c = random_cache(S, n_blocks, kv, hd, block, "int8", 11)
    tables, L = tables_for(lengths, block, n_blocks, 60).to(DEV), i32(*lengths).to(DEV)
    q = torch.randn(S, heads * hd).half().to(DEV)
    want = torch.empty_like(q)
    parts = c.parts(DEV)
    ops.attn_decode_paged(want, q, *parts, tables, L, "int8")
    wide_q, wide_out = torch.full((S, heads * hd + 24), 9.0, dtype=torch.float16, device=DEV), torch.full((S, heads * hd + 40), 9.0, dtype=torch.float16, device=DEV)
    wide_q[:, 8:8 + heads * hd] = q
    layers_k, layers_v = torch.randn(S, 3, *parts[2].shape[1:], device=DEV).half(), torch.randn(S, 3, *parts[3].shape[1:], device=DEV).half()
    layers_k[:, 1], layers_v[:, 1] = parts[2], parts[3]
    ops.attn_decode_paged(wide_out[:, 16:16 + heads * hd], wide_q[:, 8:8 + heads * hd], parts[0], parts[1], layers_k[:, 1], layers_v[:, 1], tables, L, "int8")
    assert torch.equal(wide_out[:, 16:16 + heads * hd], want) and bool((wide_out[:, :16] == 9).all()) and bool((wide_out[:, 16 + heads * hd:] == 9).all())
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.empty_like(q) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                ops.attn_decode_paged(o, q, *parts, tables, L, "int8")
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for o in outs:
        o.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.attn_decode_paged(o, q, *parts, tables, L, "int8")
        graphs.append(g)
    for _ in range(10):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    L.copy_(i32(16, 0, 299))
    graphs[0].replay()
    again = torch.empty_like(q)
    ops.attn_decode_paged(again, q, *parts, tables, L, "int8")
    assert torch.equal(outs[0], again) and bool((again[1] == 0).all()) and not torch.equal(again, want)


def test_attention_pool_beyond_32_bits():
    """Blocks whose place in the pool is beyond 2^32 bytes."""
    kv, hd, block = 8, 128, 128
    n_blocks = (1 << 32) // (kv * 2 * block * hd) + 3
    data = torch.empty(n_blocks, kv, block // 16, 2, 16 * hd, dtype=torch.uint8, device=DEV)
    scales = torch.ones(n_blocks, kv, 4, device=DEV)
    c = random_cache(1, 3, kv, hd, block, "int8", 12)
    data[-3:], scales[-3:] = c.data.to(DEV), c.scales.to(DEV)
    q, out, want = torch.randn(1, kv * hd).half().to(DEV), *(torch.empty(1, kv * hd, dtype=torch.float16, device=DEV) for _ in range(2))
    tk, tv = c.tail_k.to(DEV), c.tail_v.to(DEV)
    ids = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    ops.attn_decode_paged(want, q, c.data.to(DEV), c.scales.to(DEV), tk, tv, ids, i32(400).to(DEV), "int8")
    ops.attn_decode_paged(out, q, data, scales, tk, tv, ids + (n_blocks - 3), i32(400).to(DEV), "int8")
    assert torch.equal(out, want)
    freq, runs = inv_freq(hd).to(DEV), torch.tensor([[0, 0, 0, 128, n_blocks - 1, -1, 0, 0]], dtype=torch.int32, device=DEV)
    q, k, v = dev(*make_inputs(128, kv, kv, hd, 3))
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    ops.rope_kv_append_paged(torch.empty_like(q), q, k, v, data, scales, tk, tv, runs, one, freq, "int8")
    small, small_scales = torch.zeros_like(data[:1]), torch.zeros_like(scales[:1])
    runs[0, 4] = 0
    ops.rope_kv_append_paged(torch.empty_like(q), q, k, v, small, small_scales, tk, tv, runs, one, freq, "int8")
    assert torch.equal(data[-1], small[0]) and torch.equal(scales[-1, :, :2], small_scales[0, :, :2])


def test_paged_refusals():
    c = R.Cache(2, 4, 2, 64, 16, "int8")
    parts = list(c.parts(DEV))
    q, out = torch.zeros(2, 256, dtype=torch.float16, device=DEV), torch.zeros(2, 256, dtype=torch.float16, device=DEV)
    tables, L = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    ok = [out, q, *parts, tables, L, "int8"]
    ops.attn_decode_paged(*ok)

    def bad(i, v, match):
        with pytest.raises(RuntimeError, match=match):
            ops.attn_decode_paged(*(ok[:i] + [v] + ok[i + 1:]))
    bad(1, q.float(), "fp16 expected")
    bad(1, q[:, :192], "expected")                              # another width than out
    bad(1, q[:, :96], "expected")
    bad(1, q[:1], "expected")
    bad(1, torch.zeros(2, 512, dtype=torch.float16, device=DEV)[:, ::2], "contiguous")
    bad(1, torch.zeros(2, 260, dtype=torch.float16, device=DEV)[:, 2:258], "aligned")
    bad(2, parts[0].to(torch.int8), "Byte expected")
    bad(2, parts[0][:, :, :, :1], "expected")
    bad(3, parts[1][..., :2], "shape")
    bad(4, parts[2][:, :, :8], "shape")
    bad(5, parts[3].transpose(3, 4), "shape")
    bad(4, parts[2].transpose(1, 2).contiguous().transpose(1, 2), "contiguous")
    bad(6, tables[:, :1].t(), "shape")
    bad(7, L.long(), "Int expected")
    bad(8, "fp8", "kind")
    bad(1, q.cpu(), "CUDA tensors only")
    with pytest.raises(RuntimeError, match="workspace"):
        ops.attn_decode_paged(*ok, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError, match="must be a tensor"):
        ops.attn_decode_paged(None, *ok[1:])
    odd = R.Cache(2, 4, 2, 96, 16, "int8")                      # a head dimension without a kernel
    q96 = torch.zeros(2, 192, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="shape"):
        ops.attn_decode_paged(q96, q96, *odd.parts(DEV), tables, L, "int8")
    three = torch.zeros(2, 320, dtype=torch.float16, device=DEV)        # five heads on two
    with pytest.raises(RuntimeError, match="shape"):
        ops.attn_decode_paged(three, three, *parts, tables, L, "int8")
    q3, kv3 = torch.zeros(3, 256, dtype=torch.float16, device=DEV), torch.zeros(3, 128, dtype=torch.float16, device=DEV)
    runs, one, freq = torch.zeros(7, 8, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), inv_freq(64).to(DEV)
    fine = [q3, q3, kv3, kv3, *parts, runs, one, freq, "int8"]
    ops.rope_kv_append_paged(*fine)
    for i, v, match in ((2, kv3[:2], "expected"), (10, freq.float(), "Double expected"), (10, freq[:16], "shape"), (8, runs[:, :4], "shape"), (3, kv3[:, :64], "expected"),
                        (0, q3[:, :128], "expected")):
        with pytest.raises(RuntimeError, match=match):
            ops.rope_kv_append_paged(*(fine[:i] + [v] + fine[i + 1:]))


def test_output_rows_that_overlap_are_refused():
    c = R.Cache(2, 4, 2, 64, 16, "int8")
    parts = c.parts(DEV)
    q, one = torch.zeros(2, 256, dtype=torch.float16, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    tables, L, runs = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(5, 8, dtype=torch.int32, device=DEV)
    kv, freq = torch.zeros(2, 128, dtype=torch.float16, device=DEV), inv_freq(64).to(DEV)
    for rows in (q[:1].expand(2, 256), q.view(-1).as_strided((2, 256), (128, 1))):
        with pytest.raises(RuntimeError, match="shape"):
            ops.attn_decode_paged(rows, q, *parts, tables, L, "int8")
        with pytest.raises(RuntimeError, match="shape"):
            ops.rope_kv_append_paged(rows, q, kv, kv, *parts, runs, one, freq, "int8")
        ops.attn_decode_paged(torch.empty_like(q), rows, *parts, tables, L, "int8")                # read only: allowed
    ops.attn_decode_paged(q[:1].expand(1, 256), q[:1], parts[0], parts[1], parts[2][:1], parts[3][:1], tables[:1], L[:1], "int8")


def test_sizes_beyond_32_bits_are_refused():
    """2^32 + 4 is not 4: columns of the table (never touched), and numbers that are arguments."""
    L, out = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    runs, n = torch.zeros(4, 8, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    table = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    for at, v in ((6, 8 + (1 << 32)), (6, 8 - (1 << 32)), (7, 16 + (1 << 32)), (8, 1 + (1 << 32)), (8, 1 - (1 << 32))):
        args = [table, L, L, out, runs, n, 8, 16, 1]
        args[at] = v
        with pytest.raises(RuntimeError, match="out of range"):
            ops.kv_plan(*args)
    wide = torch.empty(1, (1 << 32) + 4, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.kv_plan(wide, L, L, out, runs, n, 8, 16, 1)
    c = R.Cache(1, 2, 1, 64, 16, "int8")
    q = torch.zeros(1, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.attn_decode_paged(q.clone(), q, *c.parts(DEV), wide, L, "int8")
