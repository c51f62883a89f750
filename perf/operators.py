"""The operators of batched decoding over a key/value cache that is held in 8 bits in blocks of tokens, and of beam search over it, as
measurable cases: plain torch forms, and (own = True) the calls of qtip_b200.ops.

A pool of blocks holds `block` tokens of one layer each; per block and key/value head there are one scale for K and one for V.  A block
is written once, when its last token arrives; until then its tokens are kept in 16 bits in the sequence's tail.

  data    (n_blocks, n_kv, block/16, 2, 16*hd) uint8   16 tokens of K, then of V, in the order below
  scales  (n_blocks, n_kv, 4) fp32                     K scale, V scale, two unused
  tail_k  (n_seqs, n_kv, block, hd) fp16               rows 0 .. length % block - 1 are in use
  tail_v  (n_seqs, n_kv, block/2, hd, 2) fp16          pairs of tokens
  tables  (n_seqs, max_blocks) int32                   the pool's block of a sequence's blocks 0 .. length / block - 1

Order of 16 tokens of K: (group of 8 tokens, half of 64 dims, token, dim).  Of V: token = 8h + 2c + e, dim = g*(hd/8) + 4n + j, in the
order (n, g, c, j, h, e).  int8: code = value / scale + 128; e4m3: the 8 bits of value / scale.
scale = max(amax, 2^-24) * fp32(1 / top), code = round(value * (top / max(amax, 2^-24))), top = 127 or 448.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TINY = 2.0 ** -24
RUN = 8          # integers of a run: sequence, first token row, first position, tokens, pool block, run of the tail, 0, 0


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a step of eight conversations: where each one's new token goes
        dict(name="plan_step", op="plan", seqs=8, block=32, max_blocks=128, n_blocks=1024, lo=0, hi=4095, new=1),
        # a large server's step that takes prompts in pieces, some sequences idle, in a pool of a whole GPU's memory
        dict(name="plan_pieces", op="plan", seqs=512, block=16, max_blocks=512, n_blocks=200000, lo=0, hi=8100, new=77),
        # the same step's append, 32 heads without sharing
        dict(name="append_step", op="append", seqs=8, heads=32, kv=32, hd=128, block=32, kind="int8", lo=100, hi=4000, new=1),
        # prompts of odd lengths, 128 query heads on 8
        dict(name="append_prompts", op="append", seqs=4, heads=128, kv=8, hd=128, block=64, kind="e4m3", lo=0, hi=0, new=2047),
        # one conversation, just begun: latency
        dict(name="attend_begun", op="attend", seqs=1, heads=32, kv=32, hd=128, block=32, kind="int8", lo=45, hi=45),
        # eight conversations of different lengths, 128 query heads on 8
        dict(name="attend_eight", op="attend", seqs=8, heads=128, kv=8, hd=128, block=32, kind="e4m3", lo=100, hi=4097),
        # one long document, 32 query heads on 8
        dict(name="attend_long", op="attend", seqs=1, heads=32, kv=8, hd=128, block=64, kind="int8", lo=131071, hi=131071),
        # a full server, 32 heads without sharing
        dict(name="attend_many", op="attend", seqs=32, heads=32, kv=32, hd=128, block=16, kind="int8", lo=1025, hi=8191),
        # one search of four beams
        dict(name="select_four", op="select", groups=1, width=4, vocab=32000, ended=0),
        # many searches of eight beams, some beams ended
        dict(name="select_many", op="select", groups=64, width=8, vocab=128256, ended=7),
        # beams over blocks: tables, tails and token logs follow their parents
        dict(name="reorder_blocks", op="reorder", groups=2, width=8, kept=4, layers=32, kv=8, hd=128, block=32, rows=128, hi=1021, dense=False),
        # beams over plain caches in 16 bits: everything follows
        dict(name="reorder_rows", op="reorder", groups=1, width=8, kept=5, layers=32, kv=8, hd=128, block=32, rows=1024, hi=1000, dense=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 32), (32, 8), (16, 1), (128, 8), (8, 8), (24, 8), (40, 8), (64, 2), (5, 5)]


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "select", "reorder"])
    block = rng.choice([16, 32, 64, 128])
    if op == "plan":
        seqs, hi = _log(rng, 1, 512), _log(rng, 1, 8000)
        new = _log(rng, 1, 300)
        mb = (hi + new) // block + 1 + rng.randrange(4)
        return dict(op=op, seqs=seqs, block=block, max_blocks=mb, n_blocks=seqs * mb + rng.randrange(5000), lo=rng.randrange(hi + 1), hi=hi, new=new)
    heads, kv = rng.choice(HEADS)
    hd, kind = rng.choice([64, 128, 128]), rng.choice(["int8", "e4m3"])
    if op == "append":
        if rng.random() < 0.5:
            hi = _log(rng, 1, 5000)
            return dict(op=op, seqs=_log(rng, 1, 128), heads=heads, kv=kv, hd=hd, block=block, kind=kind, lo=rng.randrange(hi + 1), hi=hi, new=1)
        seqs = _log(rng, 1, 16)
        # a piece of a prompt begins where a block does
        return dict(op=op, seqs=seqs, heads=heads, kv=kv, hd=hd, block=block, kind=kind, lo=0, hi=0, new=_log(rng, 2, max(4, 8000 // seqs)))
    if op == "attend":
        hi = _log(rng, 1, 131072)
        seqs = _log(rng, 1, max(1, min(256, (1 << 30) // (hi * kv * hd))))
        return dict(op=op, seqs=seqs, heads=heads, kv=kv, hd=hd, block=block, kind=kind, lo=rng.choice([0, hi // 3, hi]), hi=hi)
    if op == "select":
        width = rng.randrange(1, 17)
        vocab = _log(rng, width, 128256)
        groups = _log(rng, 1, max(1, min(64, 65000000 // (width * vocab))))
        return dict(op=op, groups=groups, width=width, vocab=vocab, ended=rng.choice([0, 0, 3]))
    width = rng.randrange(2, 17)
    dense = rng.random() < 0.5
    rows, kv = _log(rng, 8, 1024), rng.choice([1, 2, 8])
    layers = _log(rng, 1, max(1, min(32, (1 << 27) // (width * rows * kv * hd))))
    return dict(op=op, groups=_log(rng, 1, max(1, min(8, (1 << 27) // (width * layers * rows * kv * hd)))), width=width, kept=rng.randrange(1, width),
                layers=layers, kv=kv, hd=hd, block=block, rows=rows, hi=_log(rng, 1, rows if dense else rows * block), dense=dense)


def _lengths(case, seqs):
    """Lengths from lo to hi in even steps: their sum is the case's, their order the seed's."""
    lo, hi = case["lo"], case["hi"]
    return [hi] if seqs == 1 else [lo + (hi - lo) * i // (seqs - 1) for i in range(seqs)]


def _news(case, lengths):
    """New tokens: one each, or pieces of 0 to `new` (the first has it all)."""
    if case["new"] == 1:
        return [1] * len(lengths)
    if case["op"] == "append":
        return [max(1, case["new"] - 5 * i) for i in range(len(lengths))]
    return [case["new"] * ((7 * i + 4) % 5) // 4 for i in range(len(lengths))]


# ---------------------------------------------------------------------------------------------------------------- prepare
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tables(lengths, block, max_blocks, n_blocks, g):
    """Every sequence's complete blocks, anywhere in the pool."""
    ids = torch.randperm(n_blocks, generator=g, device=DEV).to(torch.int32)
    full = [n // block for n in lengths]
    cum = [0]
    for n in full:
        cum.append(cum[-1] + n)
    at = torch.tensor(cum[:-1], device=DEV)[:, None] + torch.arange(max_blocks, device=DEV)
    live = torch.arange(max_blocks, device=DEV)[None] < torch.tensor(full, device=DEV)[:, None]
    return torch.where(live, ids[at.clamp(max=max(n_blocks - 1, 0))], torch.full_like(at, -1, dtype=torch.int32)).contiguous()


def _shuffled(lengths, seed):
    lengths = list(lengths)
    random.Random(seed).shuffle(lengths)
    return lengths


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = dict(case)
    if op == "plan":
        lengths = _shuffled(_lengths(case, case["seqs"]), seed)
        new = _shuffled(_news(case, lengths), seed + 1)
        s.update(tables=_tables(lengths, case["block"], case["max_blocks"], case["n_blocks"], g))
        _add_plan(s, lengths, new)
    elif op == "append":
        block = case["block"]
        lengths = _shuffled(_lengths(case, case["seqs"]), seed)
        new = _news(case, lengths)
        mb = max(n + m for n, m in zip(lengths, new)) // block + 1
        nb = sum((n + m) // block for n, m in zip(lengths, new)) + 5
        s.update(max_new=max(new), n_blocks=nb, tables=_tables(lengths, block, mb, nb, g))
        _add_plan(s, lengths, new)
        _plan(s)
        T, kv, hd = sum(new), case["kv"], case["hd"]
        s.update(q=torch.randn(T, case["heads"] * hd, generator=g, device=DEV).half(), k=(2 * torch.randn(T, kv * hd, generator=g, device=DEV)).half(),
                 v=torch.randn(T, kv * hd, generator=g, device=DEV).half(), inv_freq=10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd))
        s["q_out"] = torch.zeros_like(s["q"])
        _add_cache(s, g, codes=False)
    elif op == "attend":
        lengths = _shuffled(_lengths(case, case["seqs"]), seed)
        mb = max(case["hi"] // case["block"], 1)
        nb = sum(n // case["block"] for n in lengths) + 3
        s.update(n_blocks=nb, tables=_tables(lengths, case["block"], mb, nb, g), lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                 q=(2 * torch.randn(case["seqs"], case["heads"] * case["hd"], generator=g, device=DEV)).half())
        s["out"] = torch.empty_like(s["q"])
        _add_cache(s, g, codes=True)
    elif op == "select":
        G, W, V = case["groups"], case["width"], case["vocab"]
        logits = 2.5 * torch.randn(G * W, V, generator=g, device=DEV)
        logits += 6.0 * (torch.rand(G * W, V, generator=g, device=DEV) < 20.0 / V)      # a few likely tokens
        s.update(logits=logits, prev_scores=-30 * torch.rand(G, W, generator=g, device=DEV), eos=2,
                 prev_tokens=torch.randint(3, max(V, 4), (G, W), generator=g, device=DEV))
        if case["ended"]:
            ended = torch.randperm(G * W, generator=g, device=DEV)[:G * W // case["ended"]]
            s["prev_tokens"].view(-1)[ended] = s["eos"]
        s.update(tokens=torch.zeros(G, W, dtype=torch.int64, device=DEV), parents=torch.zeros(G, W, dtype=torch.int32, device=DEV),
                 scores=torch.zeros(G, W, device=DEV))
    else:
        G, W = case["groups"], case["width"]
        S, L, kv, hd, block, rows = G * W, case["layers"], case["kv"], case["hd"], case["block"], case["rows"]
        s["lengths"] = torch.full((S,), case["hi"], dtype=torch.int32, device=DEV)
        r, parents = random.Random(seed), []
        for _ in range(G):                      # beams that live on keep their rows, the others follow one of them
            kept = sorted(r.sample(range(W), case["kept"]))
            parents.append([b if b in kept else r.choice(kept) for b in range(W)])
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
        half = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)  # noqa: E731
        if case["dense"]:
            s["states"] = [(half(S, L, rows, kv * hd), 1, 0), (half(S, L, rows, kv * hd), 1, 0)]
        else:
            s["states"] = [(half(S, L * kv, block, hd), 1, block), (half(S, L * kv, block // 2, 2 * hd), 2, block),
                           (torch.randint(0, 1 << 20, (S, 1, rows, 1), generator=g, device=DEV, dtype=torch.int32), block, 0),
                           (torch.randint(0, 1 << 15, (S, 1, rows * block, 1), generator=g, device=DEV), 1, 0)]
    return s


def _add_plan(s, lengths, new):
    S, T = len(lengths), sum(new)
    s.update(lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV), new=torch.tensor(new, dtype=torch.int32, device=DEV), n_tokens=T,
             lengths_out=torch.zeros(S, dtype=torch.int32, device=DEV), runs=torch.zeros(T // s["block"] + 2 * S, RUN, dtype=torch.int32, device=DEV),
             n_runs=torch.zeros(1, dtype=torch.int32, device=DEV))


def _add_cache(s, g, codes):
    S, kv, hd, block, nb = s["seqs"], s["kv"], s["hd"], s["block"], s["n_blocks"]
    shape = (nb, kv, block // 16, 2, 16 * hd)
    s["data"] = torch.zeros(shape, dtype=torch.uint8, device=DEV)
    s["scales"] = torch.zeros(nb, kv, 4, device=DEV)
    if codes:       # values that fill the 8 bits as normal ones with a largest of 3.5 deviations do
        flat = s["data"].view(-1)
        for i in range(0, flat.numel(), 1 << 28):
            part = flat[i:i + (1 << 28)]
            x = torch.randn(part.numel(), generator=g, device=DEV)
            if s["kind"] == "int8":
                part.copy_((x * 36).round().clamp(-127, 127) + 128)
            else:
                part.copy_((x * 128).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
        top = 127.0 if s["kind"] == "int8" else 448.0
        s["scales"][..., :2] = 3.5 / top * torch.exp(0.3 * torch.randn(nb, kv, 2, generator=g, device=DEV))
    s["tail_k"] = torch.randn(S, kv, block, hd, generator=g, device=DEV).half()
    s["tail_v"] = torch.randn(S, kv, block // 2, hd, 2, generator=g, device=DEV).half()


# -------------------------------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return _run_own(s)
    return {"plan": _plan, "append": _append, "attend": _attend, "select": _select, "reorder": _reorder}[s["op"]](s)


def _run_own(s):
    from qtip_b200 import ops
    op = s["op"]
    if op == "plan":
        ops.kv_plan(s["tables"], s["lengths"], s["new"], s["lengths_out"], s["runs"], s["n_runs"], s["n_blocks"], s["block"], s["n_tokens"])
        return _planned(s)
    if op == "append":
        ops.rope_kv_append_paged(s["q_out"], s["q"], s["k"], s["v"], s["data"], s["scales"], s["tail_k"], s["tail_v"], s["runs"], s["n_runs"],
                                 s["inv_freq"], s["kind"])
        return _appended(s)
    if op == "attend":
        return ops.attn_decode_paged(s["out"], s["q"], s["data"], s["scales"], s["tail_k"], s["tail_v"], s["tables"], s["lengths"], s["kind"])
    if op == "select":
        ops.beam_select(s["tokens"], s["parents"], s["scores"], s["logits"], s["prev_scores"], s["prev_tokens"], s["eos"])
        return _selected(s)
    ops.beam_reorder(s["states"], s["parents"], s["lengths"])
    return [t for t, _, _ in s["states"]]


def _planned(s):
    return dict(tables=s["tables"], lengths=s["lengths_out"], runs=s["runs"], n_runs=s["n_runs"])


def _appended(s):
    # the 8-bit codes as they are held (equal in every bit), beside the scales they are to be multiplied by
    return dict(q=s["q_out"], codes=s["data"], scales=s["scales"], tail_k=s["tail_k"], tail_v=s["tail_v"])


def _selected(s):
    return dict(tokens=s["tokens"], parents=s["parents"], scores=s["scores"])


def _plan(s):
    """Complete blocks of this step get the lowest blocks of the pool that no sequence holds, in the order of the sequences; the new
    tokens in runs, each inside one block."""
    b, tables = s["block"], s["tables"]
    S, MB = tables.shape
    L, n = s["lengths"].long(), s["new"].long()
    cu = n.cumsum(0) - n
    J = torch.arange(MB, device=DEV)
    held = torch.zeros(s["n_blocks"] + 1, dtype=torch.int32, device=DEV)
    held.scatter_(0, torch.where(J < (L // b)[:, None], tables, s["n_blocks"]).long().view(-1), 1)
    free = torch.sort(held[:-1], stable=True)[1]
    need = (L + n) // b - L // b
    base = need.cumsum(0) - need
    at = J - (L // b)[:, None]
    fresh = (at >= 0) & (at < need[:, None])
    tables.copy_(torch.where(fresh, free[(base[:, None] + at).clamp(0, s["n_blocks"] - 1)].int(), tables))
    s["lengths_out"].copy_(L + n)
    nr = torch.where(n > 0, (L + n - 1) // b - L // b + 1, 0)
    upto = nr.cumsum(0)
    r = torch.arange(s["runs"].shape[0], device=DEV)
    q = torch.searchsorted(upto, r, right=True).clamp(max=S - 1)
    i = r - (upto - nr)[q]
    pos0 = torch.where(i == 0, L[q], (L[q] // b + i) * b)
    end = torch.minimum((pos0 // b + 1) * b, (L + n)[q])
    shared = ((L % b != 0) & (nr > 1) & ((L + n) % b != 0))[q]
    block = torch.where(end % b == 0, tables[q, (pos0 // b).clamp(0, MB - 1)].long(), torch.where(shared & (i == nr[q] - 1), -2, -1))
    tail = torch.where(shared & (i == 0), upto[q] - 1, -1)
    zero = torch.zeros_like(r)
    rows = torch.stack([q, cu[q] + pos0 - L[q], pos0, end - pos0, block, tail, zero, zero], 1).int()
    s["runs"].copy_(torch.where((r < upto[-1])[:, None], rows, s["runs"]))
    s["n_runs"].copy_(upto[-1:])
    return _planned(s)


def _tokens(s):
    """Sequence and position of every new token."""
    L, n = s["lengths"].long(), s["new"].long()
    t = torch.arange(s["n_tokens"], device=DEV)
    seq = torch.searchsorted(n.cumsum(0), t, right=True)
    return seq, L[seq] + t - (n.cumsum(0) - n)[seq]


def _append(s):
    """Rotate q and k; fill up the blocks; what is complete goes to the pool in 8 bits, the rest to the tails."""
    b, kv, hd, S = s["block"], s["kv"], s["hd"], s["seqs"]
    T, half = s["n_tokens"], hd // 2
    seq, pos = _tokens(s)
    angle = pos.double()[:, None, None] * s["inv_freq"]
    cs, sn = angle.cos().float(), angle.sin().float()

    def rotate(x):
        x = x.view(T, -1, hd).float()
        x0, x1 = x[..., :half], x[..., half:]
        return torch.cat([x0 * cs - x1 * sn, x1 * cs + x0 * sn], -1).half()

    s["q_out"].copy_(rotate(s["q"]).view(T, -1))
    L, n = s["lengths"].long(), s["new"].long()
    first, end = L // b, L + n
    blocks = (s["max_new"] - 1) // b + 2
    i = torch.arange(blocks, device=DEV)
    complete = (first[:, None] + i + 1) * b <= end[:, None]
    tail_rows = torch.arange(b, device=DEV) < (end % b)[:, None]
    last = (end // b - first).clamp(max=blocks - 1)
    top = 127.0 if s["kind"] == "int8" else 448.0
    for_pool = s["tables"].gather(1, (first[:, None] + i).clamp(max=s["tables"].shape[1] - 1))[complete].long()
    for which, x, tail in ((0, rotate(s["k"]), s["tail_k"]), (1, s["v"].view(T, kv, hd), s["tail_v"])):
        rows = tail if which == 0 else tail.transpose(3, 4).reshape(S, kv, b, hd)
        buf = torch.zeros(S, blocks, kv, b, hd, dtype=torch.float16, device=DEV)
        buf[:, 0] = rows
        buf[seq, pos // b - first[seq], :, pos % b] = x
        done = buf[complete].float()                                                # (blocks, kv, b, hd)
        amax = done.abs().amax((2, 3))
        largest = amax.clamp(min=TINY)
        s["scales"][for_pool, :, which] = largest * torch.tensor(1.0 / top, device=DEV)
        code = done * torch.div(torch.full_like(largest, top), largest)[..., None, None]
        code = code.round() + 128 if s["kind"] == "int8" else code.to(torch.float8_e4m3fn).view(torch.uint8)
        code = code.to(torch.uint8).view(-1, kv, b // 16, 16, hd)
        s["data"][for_pool, :, :, which] = _pack(code, which, hd)
        kept = torch.where(tail_rows[:, None, :, None], buf[torch.arange(S, device=DEV), last], rows)
        tail.copy_(kept if which == 0 else kept.view(S, kv, b // 2, 2, hd).transpose(3, 4))
    return _appended(s)


def _pack(x, which, hd):
    """(..., 16, hd) -> (..., 16*hd) in the order of the pool."""
    lead, d = x.shape[:-2], x.dim() - 2
    if which == 0:
        x = x.reshape(*lead, 2, 8, hd // 64, 64).transpose(d + 1, d + 2)
    else:
        x = x.reshape(*lead, 2, 4, 2, 8, hd // 32, 4).permute(*range(d), d + 4, d + 3, d + 1, d + 5, d, d + 2)
    return x.reshape(*lead, 16 * hd)


def _unpack(x, which, hd):
    lead, d = x.shape[:-1], x.dim() - 1
    if which == 0:
        x = x.reshape(*lead, 2, hd // 64, 8, 64).transpose(d + 1, d + 2)
    else:
        x = x.reshape(*lead, hd // 32, 8, 4, 4, 2, 2).permute(*range(d), d + 4, d + 2, d + 5, d + 1, d, d + 3)
    return x.reshape(*lead, 16, hd)


def _attend(s):
    """softmax(q K^T / sqrt(hd)) V over each sequence's blocks and tail; zeros for a sequence without tokens."""
    b, kv, hd, S = s["block"], s["kv"], s["hd"], s["seqs"]
    MB, rep = s["tables"].shape[1], s["heads"] // kv
    ids = s["tables"].clamp(0, s["n_blocks"] - 1).long()
    full = (s["lengths"] // b).long()

    def values(which):
        x = _unpack(s["data"][ids, :, :, which], which, hd)                         # (S, MB, kv, b/16, 16, hd)
        x = x.float() - 128 if s["kind"] == "int8" else x.view(torch.float8_e4m3fn).float()
        x = x * s["scales"][ids, :, which][..., None, None, None]
        x = x.permute(0, 2, 1, 3, 4, 5).reshape(S, kv, MB * b, hd)
        tail = s["tail_k"] if which == 0 else s["tail_v"].transpose(3, 4).reshape(S, kv, b, hd)
        return torch.cat([x, tail.float()], 2)

    t = torch.arange((MB + 1) * b, device=DEV)
    seen = torch.where(t < MB * b, t < (full * b)[:, None], t - MB * b < (s["lengths"] % b)[:, None])[:, None, None]
    q = s["q"].view(S, kv, rep, hd).float()
    score = (q @ values(0).transpose(2, 3) / math.sqrt(hd)).masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    v = values(1).masked_fill(~seen.transpose(2, 3), 0.0)
    out = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"].copy_(out.view(S, -1))
    return s["out"]


def _select(s):
    """The `width` best continuations of each group: largest score + log softmax, ties to the lower beam, then the larger logit, then the
    lower token.  An ended beam has one, itself.  A parent's best one stays in its row, the others fill the rows left, in order."""
    G, W, V = s["groups"], s["width"], s["vocab"]
    x = s["logits"]
    R = min(W, V)
    best, token = torch.sort(x, dim=1, descending=True, stable=True)
    best, token = best[:, :R], token[:, :R]
    lse = torch.logsumexp(x.double(), 1).float().double()
    total = s["prev_scores"].view(-1, 1).double() + (best.double() - lse[:, None])
    ended = (s["prev_tokens"].view(-1, 1) == s["eos"])
    first = torch.arange(R, device=DEV) == 0
    total = torch.where(ended, torch.where(first, s["prev_scores"].view(-1, 1).double(), -math.inf), total)
    token = torch.where(ended, s["eos"], token)
    score, at = torch.sort(total.view(G, W * R), dim=1, descending=True, stable=True)
    score, at = score[:, :W], at[:, :W]
    parent, token = at // R, token.view(G, W * R).gather(1, at)
    beams = torch.arange(W, device=DEV)
    earlier = (parent[:, :, None] == parent[:, None, :]) & (beams[:, None] > beams[None])
    stays = ~earlier.any(2)                                                          # the best child of its parent
    taken = torch.zeros(G, W, dtype=torch.int64, device=DEV).scatter_add_(1, parent, stays.long())
    vacant = torch.sort(taken, dim=1, stable=True)[1]                                # rows without a child first, in order
    moved = (~stays).long().cumsum(1) - 1
    row = torch.where(stays, parent, vacant.gather(1, moved.clamp(min=0)))
    s["tokens"].scatter_(1, row, token)
    s["parents"].scatter_(1, row, parent.int())
    s["scores"].scatter_(1, row, score.float())
    return _selected(s)


def _reorder(s):
    """Row b of each group becomes a copy of row parents[b], as far as that one is filled."""
    G, W = s["parents"].shape
    source = (torch.arange(G, device=DEV)[:, None] * W + s["parents"]).view(-1)
    for t, per_row, mod in s["states"]:
        n = s["lengths"][source]
        n = n % mod if mod else n
        filled = torch.arange(t.shape[2], device=DEV) < ((n + per_row - 1) // per_row)[:, None]
        t.copy_(torch.where(filled[:, None, :, None], t[source], t))
    return [t for t, _, _ in s["states"]]


# ------------------------------------------------------------------------------------------------------------- work, exact
def work(case):
    op = case["op"]
    if op in ("plan", "append"):
        lengths = _lengths(case, case["seqs"])
        new = _news(case, lengths)
        # the order of the lengths is the seed's: count blocks on average
        runs = sum(max(1, n / case["block"]) for n in new if n)
        fresh = sum(new) / case["block"]
    if op == "plan":
        live = sum(n // case["block"] for n in lengths)
        return {"bytes": 4 * live + 12 * case["seqs"] + 4 * RUN * runs + 4 * fresh + 4, "flops": 0}
    if op == "append":
        T, w, kw = sum(new), case["heads"] * case["hd"], case["kv"] * case["hd"]
        done = T // case["block"] * case["block"] if case["new"] > 1 else T / case["block"]
        kept = max(0, T - done)
        # one token that completes a block: the block's other tokens are read from the tail and the whole of it is written
        rest = 0 if case["new"] > 1 else T / case["block"] * (case["block"] - 1) * kw
        return {"bytes": 4 * T * w + 4 * T * kw + 4 * kept * kw + 2 * done * kw + 4 * rest + 2 * rest + 4 * RUN * runs, "flops": 3 * T * (w + kw)}
    if op == "attend":
        lengths, b = _lengths(case, case["seqs"]), case["block"]
        full = sum(n // b for n in lengths)
        tail = sum(n % b for n in lengths)
        kw, w = case["kv"] * case["hd"], case["heads"] * case["hd"]
        return {"bytes": full * (2 * b * kw + 8 * case["kv"] + 4) + 4 * tail * kw + 4 * case["seqs"] * w, "flops": 4 * sum(lengths) * w}
    if op == "select":
        rows = case["groups"] * case["width"]
        rows -= rows // case["ended"] if case["ended"] else 0
        return {"bytes": 4 * rows * case["vocab"] + 28 * case["groups"] * case["width"], "flops": 3 * rows * case["vocab"]}
    moved, L, w, n, b = (case["width"] - case["kept"]) * case["groups"], case["layers"], case["kv"] * case["hd"], case["hi"], case["block"]
    if case["dense"]:
        one = 2 * L * n * w * 2
    else:
        one = L * w * 2 * (n % b + (n % b + 1) // 2 * 2) + 4 * ((n + b - 1) // b) + 8 * n
    return {"bytes": 2 * moved * one, "flops": 0}


def exact(case, seed):
    """Each operator from its definition, in 64 bits, a sequence or a group at a time."""
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "select":
        return _exact_select(s)
    return _exact_reorder(s) if case["op"] == "reorder" else None


def _exact_append(s):
    b, kv, hd = s["block"], s["kv"], s["hd"]
    q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    scales, tk, tv = s["scales"].double(), s["tail_k"].double(), s["tail_v"].double()
    top, t0 = (127.0 if s["kind"] == "int8" else 448.0), 0
    for i, (length, n) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
        at = torch.arange(length, length + n, device=DEV, dtype=torch.float64)
        turn = torch.exp(1j * at[:, None, None] * s["inv_freq"])

        def turned(x):
            x = x[t0:t0 + n].double().view(n, -1, 2, hd // 2)
            z = torch.complex(x[:, :, 0], x[:, :, 1]) * turn
            return torch.cat([z.real, z.imag], -1)

        q[t0:t0 + n] = turned(s["q"]).view(n, -1)
        new_k, new_v = turned(s["k"]), s["v"][t0:t0 + n].double().view(n, kv, hd)
        o = length % b
        old_v = s["tail_v"][i].double().permute(0, 1, 3, 2).reshape(kv, b, hd)
        ks = torch.cat([s["tail_k"][i].double()[:, :o], new_k.transpose(0, 1)], 1)
        vs = torch.cat([old_v[:, :o], new_v.transpose(0, 1)], 1)
        whole = (o + n) // b
        for j in range(whole):
            block = int(s["tables"][i, length // b + j])
            for w, x in ((0, ks.half().double()), (1, vs)):        # a key is the 16-bit one, as in the tail
                scales[block, :, w] = x[:, j * b:(j + 1) * b].abs().amax((1, 2)).clamp(min=TINY) / top
        rest = (o + n) % b
        if rest:
            tk[i][:, :rest] = ks[:, whole * b:]
            old_v = old_v.clone()
            old_v[:, :rest] = vs[:, whole * b:]
            tv[i] = old_v.view(kv, b // 2, 2, hd).permute(0, 1, 3, 2)
        t0 += n
    return dict(q=q, codes=None, scales=scales, tail_k=tk, tail_v=tv)


def _exact_attend(s):
    b, kv, hd, rep = s["block"], s["kv"], s["hd"], s["heads"] // s["kv"]
    t, d = torch.arange(16, device=DEV)[:, None], torch.arange(hd, device=DEV)[None]
    at_k = ((t // 8) * (hd // 64) + d // 64) * 512 + (t % 8) * 64 + d % 64
    g, n, j = d // (hd // 8), d % (hd // 8) // 4, d % 4
    at_v = (((n * 8 + g) * 4 + t % 8 // 2) * 4 + j) * 4 + (t // 8) * 2 + t % 2
    value = torch.arange(256, device=DEV, dtype=torch.uint8)
    value = value.double() - 128 if s["kind"] == "int8" else value.view(torch.float8_e4m3fn).double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, length in enumerate(s["lengths"].tolist()):
        if not length:
            continue
        ids = s["tables"][i, :length // b].long()
        both = []
        for w, at, tail in ((0, at_k, s["tail_k"][i]), (1, at_v, s["tail_v"][i].transpose(2, 3).reshape(kv, b, hd))):
            heads = []
            for h in range(kv):
                code = s["data"][ids, h, :, w]                                        # (blocks, b/16, 16*hd)
                x = value[code[..., at].long()] * s["scales"][ids, h, w].double()[:, None, None, None]
                heads.append(torch.cat([x.reshape(-1, hd), tail[h, :length % b].double()]))
            both.append(torch.stack(heads))
        q = s["q"][i].double().view(kv, rep, hd)
        p = torch.softmax(q @ both[0].transpose(1, 2) / math.sqrt(hd), -1)
        out[i] = (p @ both[1]).view(-1)
    return out


def _exact_select(s):
    G, W, V = s["groups"], s["width"], s["vocab"]
    scores = torch.zeros(G, W, dtype=torch.float64)
    rows = s["logits"].view(G, W, V)
    for g in range(G):
        found = []
        for w in range(W):
            score = float(s["prev_scores"][g, w])
            if int(s["prev_tokens"][g, w]) == s["eos"]:
                found.append((-score, w, 0))
                continue
            x = rows[g, w].double()
            part = torch.log_softmax(x, 0)
            best = torch.topk(part, min(W, V))[0].tolist()
            found += [(-(score + v), w, r) for r, v in enumerate(best)]
        found = sorted(found)[:W]
        placed, later = {}, []
        for f in found:
            if f[1] in placed:
                later.append(f)
            else:
                placed[f[1]] = f
        for f in later:
            placed[min(set(range(W)) - set(placed))] = f
        for row, f in placed.items():
            scores[g, row] = -f[0]
    return dict(tokens=None, parents=None, scores=scores.to(DEV))


def _exact_reorder(s):
    W, states = s["width"], []
    for t, per_row, mod in s["states"]:
        if not t.is_floating_point():
            states.append(None)
            continue
        out = t.double()
        for row in range(t.shape[0]):
            parent = row // W * W + int(s["parents"][row // W, row % W])
            n = int(s["lengths"][parent])
            n = -(-(n % mod if mod else n) // per_row)
            out[row, :, :n] = t[parent, :, :n].double()
        states.append(out)
    return states
