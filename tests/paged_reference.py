"""Plain restatement, on the CPU, of the 8-bit block cache and of beam search: one sequence, block, token at a time, in 64 bits where
numbers are computed."""
import math

import torch

TINY = 2.0 ** -24
TOP = {"int8": 127.0, "e4m3": 448.0}


def k_place(t, d, hd):
    """Byte of token t (of 16), dim d in a unit's K."""
    return ((t // 8) * (hd // 64) + d // 64) * 512 + (t % 8) * 64 + d % 64


def v_place(t, d, hd):
    g, n, j = d // (hd // 8), d % (hd // 8) // 4, d % 4
    return (((n * 8 + g) * 4 + t % 8 // 2) * 4 + j) * 4 + (t // 8) * 2 + t % 2


def places(which, hd):
    f = k_place if which == 0 else v_place
    return torch.tensor([[f(t, d, hd) for d in range(hd)] for t in range(16)])


def code_values(kind):
    c = torch.arange(256, dtype=torch.uint8)
    return c.double() - 128 if kind == "int8" else c.view(torch.float8_e4m3fn).double()


def quantize(x, kind):
    """x (tokens, hd) fp16 of one block and head -> codes (tokens, hd) uint8, scale, in the operator's fp32 arithmetic."""
    if not bool(torch.isfinite(x).all()):
        return torch.full(x.shape, 128 if kind == "int8" else 0, dtype=torch.uint8), float("nan")
    amax = x.float().abs().max().clamp(min=TINY).view(1)
    top = torch.tensor([TOP[kind]])
    y = x.float() * (top / amax)
    codes = (y.round() + 128).to(torch.uint8) if kind == "int8" else y.to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, float(amax * (torch.ones(1) / top))


def pack(codes, which):
    """codes (block, hd) -> bytes (block / 16, 16 * hd)."""
    block, hd = codes.shape
    out = torch.zeros(block // 16, 16 * hd, dtype=torch.uint8)
    at = places(which, hd)
    for u in range(block // 16):
        out[u][at.view(-1)] = codes[16 * u:16 * u + 16].reshape(-1)
    return out


def rotate(x, pos, inv_freq):
    """x (heads, hd) fp16 at one position: cos and sin of the 64-bit angle rounded to fp32, each product and sum rounded to fp32."""
    half = x.shape[1] // 2
    angle = float(pos) * inv_freq.double()
    cs, sn = angle.cos().float(), angle.sin().float()
    a, b = x.float()[:, :half], x.float()[:, half:]
    return torch.cat([a * cs - b * sn, b * cs + a * sn], 1).half()


def plan(tables, lengths, new, n_blocks, block, n_tokens):
    """-> tables, lengths_out, runs, status."""
    tables, S, MB = tables.clone(), tables.shape[0], tables.shape[1]
    status, held = 0, set()
    for s in range(S):
        for j in range(min(max(int(lengths[s]), 0) // block, MB)):
            if 0 <= int(tables[s, j]) < n_blocks:
                held.add(int(tables[s, j]))
            else:
                status |= 16
    free = [i for i in range(n_blocks) if i not in held]
    out, runs, row, base = [], [], 0, 0
    for s in range(S):
        L, n = int(lengths[s]), int(new[s])
        first_row = row
        row += max(n, 0)
        if L < 0 or n < 0 or L // block > MB or (L + n) // block > MB or row > n_tokens:
            status |= 1
            out.append(max(L, 0))
            continue
        need = (L + n) // block - L // block
        base += need
        if need and base > len(free):
            status |= 8
            out.append(L)
            continue
        out.append(L + n)
        mine, pos = [], L
        while pos < L + n:
            stop = min((pos // block + 1) * block, L + n)
            b = -1
            if stop % block == 0:
                b = free[base - need + pos // block - L // block]
                tables[s, pos // block] = b
            mine.append([s, first_row + pos - L, pos, stop - pos, b, -1, 0, 0])
            pos = stop
        if L % block and len(mine) > 1 and mine[-1][4] < 0:
            mine[-1][4] = -2
            mine[0][5] = len(runs) + len(mine) - 1
        runs += mine
    return tables, torch.tensor(out, dtype=torch.int32), torch.tensor(runs, dtype=torch.int32).view(-1, 8), status


class Cache:
    """The cache of one layer, on the CPU, as its parts are laid out."""

    def __init__(self, n_seqs, n_blocks, n_kv, hd, block, kind):
        self.kv, self.hd, self.block, self.kind = n_kv, hd, block, kind
        self.data = torch.zeros(n_blocks, n_kv, block // 16, 2, 16 * hd, dtype=torch.uint8)
        self.scales = torch.zeros(n_blocks, n_kv, 4)
        self.tail_k = torch.zeros(n_seqs, n_kv, block, hd).half()
        self.tail_v = torch.zeros(n_seqs, n_kv, block // 2, hd, 2).half()

    def parts(self, device):
        return tuple(t.to(device) for t in (self.data, self.scales, self.tail_k, self.tail_v))

    def append(self, s, pos, k, v, table):
        """k (n_kv, hd), already rotated, and v of one token of sequence s at position pos."""
        r = pos % self.block
        if r + 1 < self.block:
            self.tail_k[s][:, r] = k
            self.tail_v[s][:, r // 2, :, r % 2] = v
            return
        for h in range(self.kv):
            old_v = self.tail_v[s][h].permute(0, 2, 1).reshape(self.block, self.hd)
            for which, rows, last in ((0, self.tail_k[s][h], k[h]), (1, old_v, v[h])):
                x = rows.clone()
                x[r] = last
                codes, scale = quantize(x, self.kind)
                self.data[table[pos // self.block], h, :, which] = pack(codes, which)
                self.scales[table[pos // self.block], h, which] = scale

    def values(self, s, length, table, h, which):
        """(length, hd) fp64 of one head."""
        at, lut = places(which, self.hd), code_values(self.kind)
        rows = []
        for j in range(length // self.block):
            code = self.data[int(table[j]), h, :, which][:, at.view(-1)].view(-1, self.hd)
            rows.append(lut[code.long()] * float(self.scales[int(table[j]), h, which]))
        tail = self.tail_k[s, h] if which == 0 else self.tail_v[s, h].permute(0, 2, 1).reshape(self.block, self.hd)
        rows.append(tail[:length % self.block].double())
        return torch.cat(rows)

    def attend(self, q, s, length, table):
        """q (n_heads, hd) of sequence s -> (n_heads, hd) fp64."""
        if length == 0:
            return torch.zeros(q.shape, dtype=torch.float64)
        rep, out = q.shape[0] // self.kv, []
        for h in range(self.kv):
            k, v = (self.values(s, length, table, h, w) for w in (0, 1))
            p = torch.softmax(q[h * rep:(h + 1) * rep].double() @ k.T / math.sqrt(self.hd), 1)
            out.append(p @ v)
        return torch.cat(out)


def select(logits, prev_scores, prev_tokens, eos):
    """One group: logits (W, V), prev_scores, prev_tokens (W) -> tokens, parents, scores, whether there was none."""
    W, found = logits.shape[0], []
    for w in range(W):
        score = float(prev_scores[w])
        if not math.isfinite(score):
            continue
        if eos >= 0 and int(prev_tokens[w]) == eos:
            found.append((-score, w, 0, eos))
            continue
        x = logits[w].float()
        keep = torch.isfinite(x).nonzero().view(-1)
        if not len(keep):
            continue
        lse = float(torch.logsumexp(x[keep].double(), 0).float())
        order = sorted(keep.tolist(), key=lambda i: (-float(x[i]), i))[:W]
        found += [(-(score + (float(x[i]) - lse)), w, r, i) for r, i in enumerate(order)]
    found = sorted(found)[:W]
    placed, later = {}, []
    for f in found:
        if f[1] in placed:
            later.append(f)
        else:
            placed[f[1]] = f
    rows = [r for r in range(W) if r not in placed]
    for r, f in zip(rows, later):
        placed[r] = f
    tokens = [placed[r][3] if r in placed else max(eos, 0) for r in range(W)]
    parents = [placed[r][1] if r in placed else r for r in range(W)]
    scores = [-placed[r][0] if r in placed else -math.inf for r in range(W)]
    return tokens, parents, scores, not found
