"""Operators on device memory, as far as they go without a GPU: refusals of the C-ABI and the float64 oracle itself."""
import ctypes as C

import numpy as np
import pytest
import torch

import dsk
import serve_oracle as so


def _cache(**kw):
    mem = np.zeros(4096 + 16, dtype=np.uint8)
    at = (mem.ctypes.data + 15) // 16 * 16
    d = dict(k=at, v=at, k_scale=at, v_scale=at, status=None, device=0, n_blocks=4, block=16, kv_heads=2, dim_k=64, dim_v=64)
    d.update(kw)
    return dsk.Kv8(*[d[n] for n, _ in dsk.Kv8._fields_]), mem


def _rows(mem, **kw):
    at = (mem.ctypes.data + 15) // 16 * 16
    d = dict(table=at, first=at, count=None, table_pitch=2, table_blocks=2, batch=1, rows=1)
    d.update(kw)
    return dsk.Kv8Rows(*[d[n] for n, _ in dsk.Kv8Rows._fields_])


def _view(mem, **kw):
    d = dict(data=(mem.ctypes.data + 15) // 16 * 16, dtype=2, batch=128, row=128, head=64)
    d.update(kw)
    return dsk.View(*[d[n] for n, _ in dsk.View._fields_])


def _says(rc, text):
    assert rc != 0
    assert text in dsk.lib().dsk_last_error().decode(), dsk.lib().dsk_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(block=48), "16, 32, 64 or 128"), (dict(block=0), "16, 32, 64 or 128"), (dict(block=256), "16, 32, 64 or 128"), (dict(dim_k=72), "multiple of 16"), (dict(dim_v=272), "multiple of 16"),
    (dict(dim_k=0), "multiple of 16"), (dict(dim_v=-16), "multiple of 16"), (dict(kv_heads=0), "positive"), (dict(kv_heads=40000), "32767"), (dict(n_blocks=0), "positive"), (dict(k=None), "null"),
    (dict(v_scale=None), "null"), (dict(k=8 + 16 * 4096), "alignment"), (dict(k_scale=2 + 16 * 4096), "alignment"), (dict(device=-1), "CUDA device" if not torch.cuda.is_available() else "out of range"),
])
def test_cache_refusals(kw, text):
    c, mem = _cache(**kw)
    s, x = _rows(mem), _view(mem)
    L = dsk.lib()
    need = C.c_size_t()
    _says(L.dsk_kv8_write(c, s, x, x, None), text)
    _says(L.dsk_kv8_read(c, s, x, x, None), text)
    _says(L.dsk_kv8_attn_workspace(c, s, 4, 0, 0, need), text)
    _says(L.dsk_kv8_attn(c, s, x, x, 4, 1.0, 0, 0, None, 0, None), text)


@pytest.mark.parametrize("kw,text", [(dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(rows=-1), "rows"), (dict(table_blocks=-1), "blocks"), (dict(table_blocks=1 << 27), "2^30"),
                                     (dict(table=None), "null"), (dict(first=None), "null"), (dict(table_blocks=0), "empty"),
                                     (dict(table=2 + 16 * 4096), "alignment"), (dict(first=1 + 16 * 4096), "alignment"), (dict(count=2 + 16 * 4096), "alignment")])
def test_row_refusals(kw, text):
    c, mem = _cache()
    s, x = _rows(mem, **kw), _view(mem)
    L = dsk.lib()
    _says(L.dsk_kv8_write(c, s, x, x, None), text)
    _says(L.dsk_kv8_read(c, s, x, x, None), text)
    _says(L.dsk_kv8_attn(c, s, x, x, 4, 1.0, 0, 0, None, 0, None), text)


@pytest.mark.parametrize("cache,rows,view,code", [(dict(), dict(), dict(dtype=3), -4), (dict(block=48), dict(), dict(), -4), (dict(dim_v=272), dict(), dict(), -4), (dict(kv_heads=40000), dict(), dict(), -4),
                                                  (dict(), dict(batch=65536), dict(), -4), (dict(), dict(rows=-1), dict(), -4), (dict(k=None), dict(), dict(), -1), (dict(), dict(table=None), dict(), -1),
                                                  (dict(device=-1), dict(), dict(), -1)])
def test_refusals_return_their_code(cache, rows, view, code):
    """-4: a form that the call does not have, -1: memory or a device that is not there."""
    if view and not torch.cuda.is_available():
        pytest.skip("types are looked at behind the device")
    c, mem = _cache(**cache)
    s, x = _rows(mem, **rows), _view(mem, **view)
    L = dsk.lib()
    assert L.dsk_kv8_write(c, s, x, x, None) == code and L.dsk_kv8_read(c, s, x, x, None) == code
    assert L.dsk_kv8_attn(c, s, x, x, 4, 1.0, 0, 0, None, 0, None) == code
    if not view:
        assert L.dsk_kv8_attn_workspace(c, s, 4, 0, 0, C.byref(C.c_size_t())) == code


@pytest.mark.parametrize("kw,code", [(dict(batch=-1), -4), (dict(vocab=0), -4), (dict(drafts=128), -4)])
def test_verify_refusals_return_their_code(kw, code):
    d = dict(batch=1, drafts=2, vocab=8)
    d.update(kw)
    a = dsk.VerifyArgs(**d)
    assert dsk.lib().dsk_verify(a, None, 0, None) == code and dsk.lib().dsk_verify_workspace(a, C.byref(C.c_size_t())) == code


def test_null_structures():
    c, mem = _cache()
    s, x = _rows(mem), _view(mem)
    L = dsk.lib()
    _says(L.dsk_kv8_write(None, s, x, x, None), "null")
    _says(L.dsk_kv8_write(c, None, x, x, None), "null")
    _says(L.dsk_kv8_attn_workspace(c, s, 4, 0, 0, None), "bad arguments")
    _says(L.dsk_verify(None, None, 0, None), "null")
    _says(L.dsk_verify_workspace(None, C.byref(C.c_size_t())), "null")


@pytest.mark.parametrize("kw,text", [(dict(batch=-1), "batch"), (dict(drafts=-1), "drafts"), (dict(drafts=128), "drafts"), (dict(vocab=0), "vocabulary"), (dict(logits_dtype=3), "F32, F16 or BF16"),
                                     (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e-38), "2^-120"), (dict(temperature=1e-45), "2^-120"),
                                     (dict(logits=None), "null"), (dict(coins=None), "null"), (dict(draft_tokens=None), "null"), (dict(), "workspace")])
def test_verify_refusals(kw, text):
    mem = np.zeros(4096, dtype=np.uint8)
    at = mem.ctypes.data
    d = dict(logits=at, draft_probs=None, draft_tokens=at, count=None, coins=at, accepted=at, tokens=at, logits_batch=0, logits_row=0, probs_batch=0, probs_row=0, device=0, batch=1, drafts=2, vocab=8,
             logits_dtype=0, temperature=1.0)
    d.update(kw)
    _says(dsk.lib().dsk_verify(dsk.VerifyArgs(*[d[n] for n, _ in dsk.VerifyArgs._fields_]), None, 0, None), text)


def test_tensors_on_the_host_are_refused():
    with pytest.raises(dsk.DskError, match="CUDA"):
        dsk.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 2))
    z = torch.zeros(1, 1, 16, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(dsk.DskError, match="CUDA"):
        dsk.Cache8.of(z, z, torch.ones(1, 1), torch.ones(1, 1))


def test_every_source_of_the_library_makes_it_stale(monkeypatch):
    """An edit of any file that its objects depend on compiles the library again."""
    import os
    if os.environ.get("DSK_LIB") or not os.path.exists("/usr/local/cuda/bin/nvcc"):
        pytest.skip("an explicit library, or no compiler")
    dsk.build()
    folder = os.path.join(dsk.HERE, "csrc")
    made, real = [], os.path.getmtime
    monkeypatch.setattr(dsk.subprocess, "check_call", lambda *a, **k: made.append(a))
    for f in sorted(f for f in os.listdir(folder) if os.path.isfile(os.path.join(folder, f))) + ["../../include/dsk.h"]:
        new = os.path.abspath(os.path.join(folder, f))
        monkeypatch.setattr(os.path, "getmtime", lambda p: real(p) if os.path.abspath(p) != new else real(dsk.LIB_PATH) + 10)
        dsk.build()
        assert len(made) == 1, f
        made.clear()


def test_structures_have_the_compilers_layout(tmp_path):
    import os
    import subprocess
    src = tmp_path / "t.c"
    names = [("dsk_kv8", dsk.Kv8), ("dsk_kv8_rows", dsk.Kv8Rows), ("dsk_view", dsk.View), ("dsk_verify_args", dsk.VerifyArgs)]
    body = "".join(f'printf("%zu ", sizeof({c}));' + "".join(f'printf("%zu ", offsetof({c}, {n}));' for n, _ in p._fields_) for c, p in names)
    src.write_text('#include <stdio.h>\n#include "dsk.h"\nint main(void){' + body + "return 0;}")
    exe = tmp_path / "t"
    subprocess.check_call(["gcc", "-I", os.path.join(dsk.REPO, "include"), "-o", str(exe), str(src)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    want = []
    for _, p in names:
        want += [C.sizeof(p)] + [getattr(p, n).offset for n, _ in p._fields_]
    assert got == want
    assert [dsk._ROWS.size, dsk._VIEW.size, dsk._VERIFY.size] == [C.sizeof(p) for p in (dsk.Kv8Rows, dsk.View, dsk.VerifyArgs)]      # (and as the calls pack them)
    assert bytes(dsk.VerifyArgs(*range(1, 17), 0.5)) == dsk._VERIFY.pack(*range(1, 17), 0.5)
    assert bytes(dsk.Kv8Rows(*range(1, 8)))[:44] == dsk._ROWS.pack(*range(1, 8))[:44] and bytes(dsk.View(1, 2, 3, 4, 5)) == dsk._VIEW.pack(1, 2, 3, 4, 5)


# ---- the oracle ---------------------------------------------------------------------------------------------------------------------------------

def test_oracle_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(codes, so.TABLE, equal_nan=True)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.normal(size=20000) * 10.0 ** rng.uniform(-4, 2.6, size=20000), so.TABLE[:127], (so.TABLE[:126] + so.TABLE[1:127]) / 2]).astype(np.float32)
    x = np.concatenate([x, -x]).clip(-448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(so.encode(x), want)


def test_oracle_scales():
    for a in (448.0, 1.75, 3.5 * 2.0 ** -20, 1e-3, 5.0, 65504.0):
        s = so.scale_for(a)
        assert a <= 448 * s and (a > 224 * s)
    assert so.scale_for(0.0) == 2.0 ** -40 and so.scale_for(1e30) == 2.0 ** 40 and so.scale_for(1e-30) == 2.0 ** -40


def test_oracle_written_tokens_come_back_within_half_a_step():
    rng = np.random.default_rng(1)
    codes, scales = np.zeros((4, 2, 16, 16), dtype=np.uint8), np.ones((4, 2))
    x = rng.normal(size=(1, 40, 2, 16)) * np.exp(rng.normal(size=(1, 40, 2, 1)))
    table = np.array([[2, 0, 3]])
    for lo, hi in ((0, 5), (5, 6), (6, 33), (33, 40)):
        so.write(codes, scales, table, [lo], [hi - lo], x[:, lo:hi])
    for h in range(2):
        got, there = so.gather(codes, scales, table[0], 40, h)
        assert there.all()
        step = np.abs(x[0, :, h]) * 2.0 ** -4 + 2.0 ** -10 * scales[table[0][np.arange(40) // 16], h][:, None]
        assert (np.abs(got - x[0, :, h]) <= 2 * step).all()         # rounded twice at most


def test_oracle_attention_of_one_block_is_a_softmax():
    rng = np.random.default_rng(2)
    k, v = (rng.integers(0, 120, size=(1, 1, 16, 16)).astype(np.uint8) for _ in range(2))
    q = rng.normal(size=(1, 2, 2, 16))
    out, _, _, _ = so.attend(k, np.ones((1, 1)), v, np.ones((1, 1)), [[0]], [10], [2], q, 2, 0.01)
    for i, t in ((0, 8), (1, 9)):
        for h in range(2):
            w = np.exp(so.TABLE[k[0, 0, :t + 1]] @ q[0, i, h] * 0.01)
            assert np.allclose(out[0, i, h], w @ so.TABLE[v[0, 0, :t + 1]] / w.sum(), rtol=1e-12)


def test_oracle_verification_draws_from_the_target():
    """Whatever the draft model says, the first token of a verification is distributed as the target's: 20000 runs, standard deviations of the counts."""
    rng = np.random.default_rng(3)
    V, N = 5, 20000
    logits = np.repeat(rng.normal(size=(1, 2, V)), N, 0)
    q = rng.dirichlet(np.ones(V))
    drafts = rng.choice(V, size=(N, 1), p=q)
    acc, tok = so.verify(logits, drafts, rng.random((N, 2)), np.broadcast_to(q, (N, 1, V)), np.ones(N, dtype=int), 1.0)
    p = np.exp(logits[0, 0])
    p /= p.sum()
    got = np.bincount(tok[:, 0], minlength=V)
    assert (np.abs(got - N * p) <= 5 * np.sqrt(N * p * (1 - p))).all()
