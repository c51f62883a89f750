"""CPU: the new entry points refuse what their documentation rules out before touching a device, and the layout's formulas are one to one."""
import ctypes

import pytest
import torch

import paged_reference as R
from qtip_b200 import _lib, ops

P = (ctypes.addressof(ctypes.create_string_buffer(4096)) + 255) & ~255


def test_plan_arguments():
    f = _lib.load().qtip_kv_plan
    ok = [P, P + 16, P + 32, P + 48, P + 64, P + 128, 2, 4, 8, 16, 3, 4, None, None]

    def st(i, v):
        return f(*(ok[:i] + [v] + ok[i + 1:]))
    for i in range(6):
        assert st(i, None) == _lib.ERR_BAD_ARG
    assert st(3, P + 16) == _lib.ERR_BAD_ARG and st(3, P + 32) == _lib.ERR_BAD_ARG
    for i, v in ((6, 0), (6, 65536), (7, 0), (8, 0), (8, 1600001), (9, 8), (9, 48), (9, 256), (10, -1), (10, (1 << 20) + 1), (7, 1 << 27)):
        assert st(i, v) == _lib.ERR_BAD_SHAPE, (i, v)
    assert st(11, 3) == _lib.ERR_WORKSPACE
    assert st(4, P + 68) == _lib.ERR_ALIGNMENT and st(0, P + 2) == _lib.ERR_ALIGNMENT and st(12, P + 1) == _lib.ERR_ALIGNMENT


def test_append_arguments():
    f = _lib.load().qtip_rope_kv_append_paged
    #     q_out      q      k      v      data scales tail_k     tail_v     runs n_runs max inv_freq T  S  H  kv hd  nb blk kind
    ok = [P, 64, P, 64, P, 64, P, 64, P, P, P, 2048, P, 2048, P, P, 4, P, 2, 2, 1, 1, 64, 4, 16, 0, None, None]

    def st(i, v):
        return f(*(ok[:i] + [v] + ok[i + 1:]))
    for i in (0, 2, 4, 6, 8, 9, 10, 12, 14, 15, 17):
        assert st(i, None) == _lib.ERR_BAD_ARG
    for i, v in ((16, -1), (18, -1), (19, 0), (20, 0), (21, 0), (22, 96), (22, 256), (23, 0), (24, 24), (24, 8), (25, 2), (25, -1)):
        assert st(i, v) == _lib.ERR_BAD_SHAPE, (i, v)
    for i, v in ((0, P + 8), (2, P + 2), (8, P + 8), (14, P + 4), (1, 68), (3, 65), (11, 2052), (17, P + 4), (15, P + 2)):
        assert st(i, v) == _lib.ERR_ALIGNMENT, (i, v)
    assert st(18, 0) == _lib.OK and st(16, 0) == _lib.OK          # nothing to do


def test_attention_arguments():
    lib = _lib.load()
    need = lib.qtip_attn_paged_workspace_bytes(2, 8, 2, 64)
    assert need > 0 and lib.qtip_attn_paged_workspace_bytes(0, 8, 2, 64) == 0 and lib.qtip_attn_paged_workspace_bytes(2, 8, 3, 64) == 0
    f = lib.qtip_attn_decode_paged
    #     out     q       data scales tail_k  tail_v  tables lengths S H kv hd mb nb blk kind ws
    ok = [P, 512, P, 512, P, P, P, 2048, P, 2048, P, P, 2, 8, 2, 64, 4, 8, 16, 0, P, need, None, None]

    def st(i, v):
        return f(*(ok[:i] + [v] + ok[i + 1:]))
    for i in (0, 2, 4, 5, 6, 8, 10, 11):
        assert st(i, None) == _lib.ERR_BAD_ARG
    for i, v in ((12, 0), (12, 65536), (13, 7), (14, 0), (15, 32), (16, 0), (16, 1 << 27), (17, 0), (18, 20), (19, 2)):
        assert st(i, v) == _lib.ERR_BAD_SHAPE, (i, v)
    assert st(20, None) == _lib.ERR_WORKSPACE and st(21, need - 1) == _lib.ERR_WORKSPACE
    for i, v in ((0, P + 8), (2, P + 4), (6, P + 8), (20, P + 4), (1, 516), (3, 513), (9, 2050), (10, P + 2), (11, P + 1)):
        assert st(i, v) == _lib.ERR_ALIGNMENT, (i, v)
    big = lib.qtip_attn_paged_workspace_bytes(65535, 8, 2, 64)
    assert f(*(ok[:12] + [65535, 8, 2, 64, 1 << 20, 8, 16, 0, P, big, None, None])) == _lib.ERR_TOO_LARGE


def test_rows_that_overlap_are_refused():
    """Rows that are written: a stride below their width would have several CTAs write one place."""
    lib = _lib.load()
    append = [P, 128, P, 128, P, 64, P, 64, P, P, P, 1024, P, 1024, P, P, 4, P, 2, 2, 2, 1, 64, 4, 16, 0, None, None]
    need = lib.qtip_attn_paged_workspace_bytes(2, 8, 2, 64)
    attend = [P, 512, P, 512, P, P, P, 2048, P, 2048, P, P, 2, 8, 2, 64, 4, 8, 16, 0, P, need, None, None]
    for f, ok, at, width in ((lib.qtip_rope_kv_append_paged, append, 1, 128), (lib.qtip_rope_kv_append_paged, append, 11, 1024),
                             (lib.qtip_rope_kv_append_paged, append, 13, 1024), (lib.qtip_attn_decode_paged, attend, 1, 512)):
        for stride in (0, 8, width - 8, -width):
            assert f(*(ok[:at] + [stride] + ok[at + 1:])) == _lib.ERR_BAD_SHAPE, (at, stride)


def test_beam_arguments():
    lib = _lib.load()
    ok = [P, P, P, P, _lib.F32, 100, P, P, 2, 4, 100, -1, None, None]

    def st(i, v):
        return lib.qtip_beam_select(*(ok[:i] + [v] + ok[i + 1:]))
    for i in (0, 1, 2, 3, 6):
        assert st(i, None) == _lib.ERR_BAD_ARG
    assert st(4, _lib.F16_FRAGMENTS) == _lib.ERR_BAD_ARG
    assert lib.qtip_beam_select(*(ok[:7] + [None] + ok[8:11] + [2, None, None])) == _lib.ERR_BAD_ARG       # eos without tokens
    for i, v in ((8, 0), (8, 65536), (9, 0), (9, 17), (10, 0), (5, 99), (10, (1 << 30) + 1)):
        assert st(i, v) == _lib.ERR_BAD_SHAPE, (i, v)

    for i, v in ((0, P + 4), (1, P + 2), (2, P + 1), (3, P + 2), (6, P + 2), (7, P + 4), (12, P + 2)):
        assert st(i, v) == _lib.ERR_ALIGNMENT, (i, v)

    def reorder(n=1, parents=P, groups=1, width=2, **kw):
        state = dict(base=P, seq_stride=64, outer_stride=64, outer=1, rows=2, row_bytes=32, per_row=1, mod=0, **{})
        state.update(kw)
        arr = (_lib.BeamState * 9)(*[_lib.BeamState(**state)] * 9)
        return lib.qtip_beam_reorder(arr, n, parents, None, groups, width, None, None)
    assert reorder(n=0) == _lib.ERR_BAD_ARG and reorder(n=9) == _lib.ERR_BAD_ARG and reorder(parents=None) == _lib.ERR_BAD_ARG and reorder(base=None) == _lib.ERR_BAD_ARG
    for kw in (dict(groups=0), dict(width=17), dict(outer=0), dict(rows=0), dict(row_bytes=2), dict(row_bytes=30), dict(per_row=0), dict(mod=-1), dict(seq_stride=60),
               dict(seq_stride=66), dict(outer=2), dict(outer=2, seq_stride=128, outer_stride=32), dict(outer=2, seq_stride=128, outer_stride=66)):
        assert reorder(**kw) == _lib.ERR_BAD_SHAPE, kw
    assert reorder(base=P + 2) == _lib.ERR_ALIGNMENT and reorder(parents=P + 2) == _lib.ERR_ALIGNMENT
    assert reorder(n=2) == _lib.ERR_BAD_ARG                       # the same state twice
    assert reorder(rows=1 << 28, seq_stride=1 << 34) == _lib.ERR_TOO_LARGE
    assert reorder(width=1) == _lib.OK                            # a beam alone has nowhere to go


def test_reorder_refuses_to_reorder_what_it_reads():
    """Parents or lengths inside a state: some CTAs would read them before, others after the copy."""
    f = _lib.load().qtip_beam_reorder

    def st(base, parents, lengths, n=1, **kw):
        state = dict(dict(seq_stride=8, outer_stride=8, outer=1, rows=1, row_bytes=4, per_row=1, mod=0), **kw)
        states = [_lib.BeamState(base=P + 2048, **state), _lib.BeamState(base=base, **state)][2 - n:]
        return f((_lib.BeamState * n)(*states), n, parents, lengths, 2, 2, None, None)
    # 2 groups of 2: 16 bytes of either; a state of 4 sequences, 8 bytes apart: 28 bytes
    for at in (P + 1024, P + 1024 - 12, P + 1024 + 24, P + 1024 + 8):
        for n in (1, 2):
            assert st(P + 1024, at, None, n) == _lib.ERR_BAD_ARG and st(P + 1024, P, at, n) == _lib.ERR_BAD_ARG
    assert st(P + 1024, P, P + 1024 + 40, outer=2, seq_stride=24, outer_stride=12) == _lib.ERR_BAD_ARG
    assert st(P + 1024, P + 1024, None, rows=0) == _lib.ERR_BAD_SHAPE


@pytest.mark.parametrize("hd", [64, 128])
def test_places_in_a_unit(hd):
    for which in (0, 1):
        assert sorted(R.places(which, hd).view(-1).tolist()) == list(range(16 * hd))


def test_wrappers_refuse_host_tensors():
    t = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.kv_plan(t, t[0], t[1], t[0], torch.zeros(6, 8, dtype=torch.int32), t[0, :1], 4, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.beam_select(t.long(), t, t.float(), torch.zeros(4, 9), t.float())
    with pytest.raises(RuntimeError, match="must be a tensor"):
        ops.beam_reorder([], None)
    with pytest.raises(RuntimeError, match="kind"):
        ops.attn_decode_paged(t, t, t, t, t, t, t, t, "int4")
