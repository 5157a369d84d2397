"""Operators on packed rows, as far as they go without a GPU: refusals of the C-ABI, structures, and the float64 oracle itself."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import dsk
import packed_oracle as po

MEM = np.zeros(4096 + 16, dtype=np.uint8)
AT = (MEM.ctypes.data + 15) // 16 * 16


def blocks(**kw):
    d = dict(free=AT, n_free=AT, status=None, device=0, n_blocks=4, block=16)
    d.update(kw)
    return dsk.BlocksArgs(*[d[n] for n, _ in dsk.BlocksArgs._fields_])


def packed(**kw):
    d = dict(starts=AT, lens=AT + 1024, positions=AT, slots=AT, pieces=AT, status=None, rows=8, batch=2, n_pieces=8, block=16, device=0)
    d.update(kw)
    return dsk.PackedArgs(*[d[n] for n, _ in dsk.PackedArgs._fields_])


def view(**kw):
    d = dict(data=AT, dtype=2, batch=0, row=128, head=64)
    d.update(kw)
    return dsk.View(*[d[n] for n, _ in dsk.View._fields_])


def cache(**kw):
    d = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, status=None, device=0, n_blocks=4, block=16, kv_heads=2, dim_k=64, dim_v=64)
    d.update(kw)
    return dsk.Kv8(*[d[n] for n, _ in dsk.Kv8._fields_])


def says(rc, text, code=None):
    assert rc != 0 and (code is None or rc == code), rc
    assert text in dsk.lib().dsk_last_error().decode(), dsk.lib().dsk_last_error()


NO_GPU = "CUDA device" if not torch.cuda.is_available() else "out of range"


@pytest.mark.parametrize("kw,text,code", [
    (dict(block=48), "16, 32, 64 or 128", -4), (dict(n_blocks=0), "at least one", -4), (dict(n_blocks=1 << 27), "2^31", -4), (dict(free=None), "null", -1), (dict(n_free=None), "null", -1),
    (dict(free=AT + 2), "alignment", -1), (dict(status=AT + 1), "alignment", -1), (dict(device=-1), NO_GPU, -1)])
def test_pool_refusals(kw, text, code):
    L, b = dsk.lib(), blocks(**kw)
    says(L.dsk_blocks_cut(b, AT, 4, 4, AT, AT, 2, None), text, code)
    says(L.dsk_blocks_extend(b, AT, 4, 4, AT, AT, packed(block=kw.get("block", 16)), None), text, code)


@pytest.mark.parametrize("table,pitch,width,batch,text,code", [
    (None, 4, 4, 2, "table", -1), (AT + 2, 4, 4, 2, "table", -1), (AT, 4, 0, 2, "table", -1), (AT, 3, 4, 2, "overlap", -4), (AT, 4, 1 << 27, 2, "2^30", -4), (AT, 4, -1, 2, "2^30", -4),
    (AT, 4, 4, -1, "sequences", -4), (AT, 4, 4, 1025, "1024", -4)])
def test_table_refusals(table, pitch, width, batch, text, code):
    L = dsk.lib()
    says(L.dsk_blocks_cut(blocks(), table, pitch, width, AT, AT, batch, None), text, code)
    says(L.dsk_blocks_extend(blocks(), table, pitch, width, AT, AT, packed(batch=batch), None), text, code)


@pytest.mark.parametrize("kw,text,code", [
    (dict(rows=-1), "packed rows", -4), (dict(rows=(1 << 20) + 1), "2^20", -4), (dict(starts=None), "starts", -1), (dict(starts=AT + 2), "starts", -1), (dict(block=32), "blocks of 32", -4),
    (dict(n_pieces=3), "pieces", -4), (dict(pieces=None), "pieces", -1), (dict(pieces=AT + 8), "16-byte", -1), (dict(lens=None), "lengths", -1), (dict(lens=AT + 4), "old ones", -1),
    (dict(positions=None), "positions", -1), (dict(slots=AT + 2), "slots", -1), (dict(status=AT + 2), "starts", -1)])
def test_packed_refusals(kw, text, code):
    says(dsk.lib().dsk_blocks_extend(blocks(), AT, 4, 4, AT, AT + 512, packed(**kw), None), text, code)


def test_extend_refuses_lengths_over_counts_and_null_structures():
    L = dsk.lib()
    says(L.dsk_blocks_extend(blocks(), AT, 4, 4, AT, AT + 1024, packed(), None), "counts", -1)
    says(L.dsk_blocks_extend(blocks(), AT, 4, 4, None, AT, packed(), None), "lengths", -1)
    says(L.dsk_blocks_extend(None, AT, 4, 4, AT, AT, packed(), None), "null", -1)
    says(L.dsk_blocks_extend(blocks(), AT, 4, 4, AT, AT, None, None), "null", -1)
    says(L.dsk_blocks_cut(None, AT, 4, 4, AT, AT, 2, None), "null", -1)
    says(L.dsk_blocks_cut(blocks(), AT, 4, 4, AT, None, 2, None), "lengths", -1)
    assert L.dsk_blocks_cut(blocks(), None, 0, 0, None, None, 0, None) == 0          # no sequence: nothing to do


@pytest.mark.parametrize("kw,plan,v,text,code", [
    (dict(dim_k=72), {}, {}, "multiple of 16", -4), (dict(k=None), {}, {}, "null", -1), (dict(block=32), {}, {}, "a cache of 32", -4), (dict(), dict(pieces=None), {}, "pieces", -1),
    (dict(), dict(n_pieces=2), {}, "pieces", -4), (dict(), dict(batch=2000), {}, "1024", -4), (dict(), {}, dict(dtype=3), "F32, F16 or BF16", -4), (dict(), {}, dict(data=None), "null", -1),
    (dict(), {}, dict(data=AT + 1), "aligned", -1), (dict(device=-1), {}, {}, NO_GPU, -1)])
def test_append_refusals(kw, plan, v, text, code):
    says(dsk.lib().dsk_kv8_append(cache(**kw), packed(**plan), view(**v), view(**v), None), text, code)


def test_append_of_nothing():
    L = dsk.lib()
    assert L.dsk_kv8_append(cache(), packed(rows=0, n_pieces=0, pieces=None), view(), view(), None) == 0
    says(L.dsk_kv8_append(None, packed(), view(), view(), None), "null", -1)
    says(L.dsk_kv8_append(cache(), None, view(), view(), None), "null", -1)
    says(L.dsk_kv8_append(cache(), packed(), None, view(), None), "F32, F16 or BF16", -4)


def attend(plan=None, q=None, k=None, v=None, o=None, heads=2, kv=1, dk=64, dv=64, scale=1.0, window=0, keep=0):
    V = lambda x: view(**(x or {}))
    return dsk.lib().dsk_packed_attn(packed(**(plan or {})), V(q), V(k), V(v), V(o), heads, kv, dk, dv, scale, window, keep, None)


@pytest.mark.parametrize("kw,text,code", [
    (dict(q=dict(dtype=0)), "F16 or BF16", -4), (dict(k=dict(dtype=1)), "keys", -4), (dict(v=dict(dtype=0)), "values", -4), (dict(o=dict(dtype=1)), "output", -4), (dict(q=dict(data=None)), "null", -1),
    (dict(o=dict(data=None)), "null", -1), (dict(dk=72), "multiple of 16", -4), (dict(dv=272), "multiple of 16", -4), (dict(dk=0), "multiple of 16", -4), (dict(heads=3, kv=2), "multiple", -4),
    (dict(heads=0), "multiple", -4), (dict(kv=0), "multiple", -4), (dict(heads=40000), "32767", -4), (dict(scale=-0.5), "not negative", -4), (dict(scale=float("inf")), "not negative", -4),
    (dict(scale=float("nan")), "not negative", -4), (dict(window=-1), "negative", -4), (dict(keep=-1), "negative", -4), (dict(q=dict(data=AT + 8)), "16-byte", -4), (dict(k=dict(data=AT + 2)), "16-byte", -4),
    (dict(q=dict(head=60)), "multiple of 8", -4), (dict(v=dict(row=0)), "multiple of 8", -4), (dict(k=dict(row=-64)), "multiple of 8", -4), (dict(plan=dict(batch=1025)), "1024", -4),
    (dict(plan=dict(rows=1 << 21)), "2^20", -4), (dict(plan=dict(starts=None)), "starts", -1), (dict(plan=dict(device=-1)), NO_GPU, -1)])
def test_attention_refusals(kw, text, code):
    says(attend(**kw), text, code)


def test_attention_over_nothing():
    assert attend(plan=dict(batch=0)) == 0 and attend(plan=dict(rows=0), q=dict(data=None)) == 0
    says(dsk.lib().dsk_packed_attn(None, view(), view(), view(), view(), 1, 1, 64, 64, 1.0, 0, 0, None), "null", -1)


def test_tensors_on_the_host_are_refused():
    z = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: dsk.Packed.of(z, 5), lambda: dsk.Blocks.of(z, 5)):
        with pytest.raises(dsk.DskError, match="CUDA"):
            call()


def test_structures_have_the_compilers_layout(tmp_path):
    src, exe = tmp_path / "t.c", tmp_path / "t"
    names = [("dsk_blocks", dsk.BlocksArgs), ("dsk_packed", dsk.PackedArgs)]
    body = "".join(f'printf("%zu ", sizeof({c}));' + "".join(f'printf("%zu ", offsetof({c}, {n}));' for n, _ in p._fields_) for c, p in names)
    src.write_text('#include <stdio.h>\n#include "dsk.h"\nint main(void){' + body + "return 0;}")
    subprocess.check_call(["gcc", "-I", os.path.join(dsk.REPO, "include"), "-o", str(exe), str(src)])
    want = []
    for _, p in names:
        want += [C.sizeof(p)] + [getattr(p, n).offset for n, _ in p._fields_]
    assert [int(v) for v in subprocess.check_output([str(exe)]).split()] == want
    assert dsk._PACKED.size == C.sizeof(dsk.PackedArgs) and bytes(dsk.PackedArgs(*range(1, 12)))[:68] == dsk._PACKED.pack(*range(1, 12))[:68]


# ---- the oracle ---------------------------------------------------------------------------------------------------------------------------------

def test_oracle_places_are_disjoint_and_come_back():
    rng = np.random.default_rng(0)
    free, table, lens = list(rng.permutation(40)), np.full((5, 9), -1), [0] * 5
    before = list(free)
    for step in range(4):
        starts, new, positions, slots, pieces, status = po.extend(free, table, lens, [3, 0, 17, 1, 20], 60, 40, 16)
        assert status == 0 and new == [l + c for l, c in zip(lens, [3, 0, 17, 1, 20])] and starts == [0, 3, 3, 20, 21, 41]
        assert positions[:3] == [lens[0] + i for i in range(3)] and positions[41:] == [-1] * 19
        assert sum(p[1] for p in pieces) == 41 and len(pieces) <= min(60, 60 // 16 + 2 * 5)
        lens = new
        held = [int(x) for b in range(5) for x in table[b, :-(-lens[b] // 16)]]
        assert sorted(held + free) == list(range(40))
    assert po.cut(free, table, lens, [0] * 5, 40, 16) == 0 and (table == -1).all() and sorted(free) == sorted(before)


def test_oracle_bound_of_pieces_holds():
    rng = np.random.default_rng(1)
    for _ in range(300):
        block, B = int(rng.choice([16, 32, 64, 128])), int(rng.integers(1, 9))
        lens, count = ([int(x) for x in rng.integers(0, n, size=B)] for n in (200, rng.choice([2, 4, 40, 300])))
        rows, table = sum(count), np.full((B, 40), 0)
        pieces = po.extend([0] * 400, table, lens, count, rows, 1, block)[4]
        assert len(pieces) <= min(rows, rows // block + 2 * B)


def test_oracle_attention_is_a_softmax():
    rng = np.random.default_rng(2)
    q, k, v = rng.normal(size=(9, 2, 16)), rng.normal(size=(9, 1, 16)), rng.normal(size=(9, 1, 32))
    out, mass, size, top = po.attend(q, k, v, [1, 6, 8], 0.3, window=3, keep=1)
    assert np.isnan(out[0]).all() and np.isnan(out[8]).all()
    for row, keys in ((1, [1]), (4, [1, 2, 3, 4]), (5, [1, 3, 4, 5]), (7, [6, 7])):
        for h in range(2):
            w = np.exp(k[keys, 0] @ q[row, h] * 0.3)
            assert np.allclose(out[row, h], w @ v[keys, 0] / w.sum(), rtol=1e-12) and (mass[row, h] >= np.abs(out[row, h])).all()
