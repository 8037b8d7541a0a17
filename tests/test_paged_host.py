"""Paged KV cache entry points without a device: struct layouts, the refusals
of the C ABI (host checks only; the pointers are placeholders that nothing
dereferences) and of the Python wrappers, and the oracle's own page plan."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from dforktree_b200 import _lib as L
from dforktree_b200 import kernels as K
from oracle import paged as OP

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x10000


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        from dforktree_b200 import build
        build.build()
    return L.load()


STRUCTS = {"dft_page_plan_args": L.PagePlanArgs, "dft_kv_append_args": L.KvAppendArgs,
           "dft_kv_commit_args": L.KvCommitArgs, "dft_chunk_attn_args": L.ChunkAttnArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "dforktree_b200.h"', 'int main(void) {']
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} SIZE %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    r = subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "p")],
                       capture_output=True, text=True)
    if r.returncode != 0:
        pytest.skip("gcc unavailable: " + r.stderr[:200])
    for line in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, val = line.split()
        got = ctypes.sizeof(STRUCTS[name]) if field == "SIZE" else getattr(STRUCTS[name], field).offset
        assert got == int(val), (name, field)


@pytest.mark.parametrize("call", [K._PAGE_PLAN, K._KV_APPEND, K._KV_COMMIT, K._CHUNK_ATTN], ids=lambda c: c.name)
def test_packed_fields_are_the_struct(call):
    v = [3.5 if t is L.f32 else 1 << 20 | i for i, (_, t) in enumerate(call.cls._fields_)]
    assert call.pack(*v) == bytes(call.cls(*v))


def _plan(**kw):
    d = dict(B=2, page_size=16, cached=FAKE, fresh=FAKE, rows=None, block_table=FAKE, bt_sr=8, n_rows=4, max_pages=8,
             held=FAKE, free_pages=FAKE, n_free=FAKE, n_pages=32, qo_indptr=FAKE, kv_indptr=FAKE, kv_indices=FAKE,
             kv_capacity=100, slot_map=FAKE, positions=FAKE, token_capacity=10)
    d.update(kw)
    return L.PagePlanArgs(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(B=-1), 1), (dict(page_size=0), 1), (dict(page_size=12), 1), (dict(page_size=-16), 1), (dict(cached=None), 1),
    (dict(held=None), 1), (dict(block_table=None), 1), (dict(free_pages=None), 1), (dict(n_free=None), 1),
    (dict(qo_indptr=None), 1), (dict(kv_indices=None), 1), (dict(slot_map=None), 1), (dict(positions=None), 1),
    (dict(bt_sr=7), 1), (dict(kv_capacity=-1), 1), (dict(B=1025), 2), (dict(page_size=2048), 2),
    (dict(n_pages=1 << 27, page_size=16), 2), (dict(max_pages=1 << 27, bt_sr=1 << 27, page_size=16), 2),
])
def test_page_plan_refuses(lib, kw, rc):
    assert lib.dft_page_plan(ctypes.byref(_plan(**kw)), None, None) == rc


def _append(**kw):
    d = dict(T=4, Hkv=2, D=64, dtype=L.DFT_BF16, k=FAKE, k_st=128, k_sh=64, v=FAKE, v_st=128, v_sh=64, k_cache=FAKE,
             v_cache=FAKE, kv_st=128, kv_sh=64, n_slots=10, slot_map=FAKE)
    d.update(kw)
    return L.KvAppendArgs(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(T=-1), 1), (dict(Hkv=0), 1), (dict(D=0), 1), (dict(dtype=L.DFT_F32), 1), (dict(dtype=9), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(k_cache=None), 1), (dict(slot_map=None), 1), (dict(k=FAKE + 1), 1),
    (dict(Hkv=1 << 20, D=1 << 10), 2), (dict(T=0, k=None, v=None, slot_map=None), 0),
])
def test_kv_append_refuses(lib, kw, rc):
    assert lib.dft_kv_append(ctypes.byref(_append(**kw)), None, None) == rc


def _commit(**kw):
    d = dict(L=1, B=2, N=32, P=24, Hkv=2, D=64, dtype=L.DFT_BF16, k_cache=FAKE, v_cache=FAKE, kv_sl=1280, kv_st=128,
             kv_sh=64, n_slots=10, kv_indptr=FAKE, kv_indices=FAKE, n_kv=100, path=FAKE, accept_len=FAKE)
    d.update(kw)
    return L.KvCommitArgs(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(L=-1), 1), (dict(B=-1), 1), (dict(N=0), 1), (dict(P=-1), 1), (dict(dtype=L.DFT_F32), 1), (dict(path=None), 1),
    (dict(accept_len=None), 1), (dict(kv_indptr=None), 1), (dict(kv_indices=None), 1), (dict(n_kv=-1), 1),
    (dict(N=65), 2), (dict(L=65536), 2), (dict(B=0), 0), (dict(P=0), 0), (dict(L=0), 0),
])
def test_kv_commit_refuses(lib, kw, rc):
    assert lib.dft_kv_commit(ctypes.byref(_commit(**kw)), None, None) == rc


def _attn(**kw):
    d = dict(B=2, T=4, Hq=8, Hkv=2, D=64, dtype=L.DFT_BF16, q=FAKE, q_st=512, q_sh=64, k_cache=FAKE, v_cache=FAKE,
             kv_st=128, kv_sh=64, n_slots=10, qo_indptr=FAKE, kv_indptr=FAKE, kv_indices=FAKE, n_kv=10,
             sm_scale=0.125, o=FAKE, o_st=512, o_sh=64)
    d.update(kw)
    return L.ChunkAttnArgs(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(B=-1), 1), (dict(T=-1), 1), (dict(Hq=7), 1), (dict(Hkv=0), 1), (dict(dtype=L.DFT_F32), 1),
    (dict(sm_scale=0.0), 1), (dict(sm_scale=-1.0), 1), (dict(sm_scale=float("nan")), 1),
    (dict(sm_scale=float("inf")), 1), (dict(q=None), 1), (dict(o=None), 1), (dict(k_cache=None), 1),
    (dict(kv_indices=None), 1), (dict(n_kv=-1), 1), (dict(D=96), 2), (dict(D=512), 2), (dict(B=1025), 2),
    (dict(Hq=258), 2), (dict(q=FAKE + 8), 2), (dict(q_st=516), 2), (dict(kv_sh=60), 2), (dict(o_st=513), 2),
])
def test_chunk_attn_refuses(lib, kw, rc):
    a = _attn(**kw)
    assert lib.dft_chunk_attn_workspace_bytes(ctypes.byref(a)) == -1
    assert lib.dft_chunk_attn(ctypes.byref(a), FAKE, None, None) == rc


def test_null_arguments_and_empty_calls(lib):
    for f, n in (("dft_page_plan", 3), ("dft_kv_append", 3), ("dft_kv_commit", 3), ("dft_chunk_attn", 4)):
        assert getattr(lib, f)(*[None] * n) == 1
    assert lib.dft_chunk_attn_workspace_bytes(None) == -1
    assert lib.dft_chunk_attn(ctypes.byref(_attn(T=0, q=None, o=None)), None, None, None) == 0
    assert lib.dft_chunk_attn(ctypes.byref(_attn(B=0, q=None, o=None)), None, None, None) == 0


def test_wrappers_refuse_shapes_before_any_device_work():
    bf = torch.bfloat16
    q, k = torch.zeros(4, 8, 64, dtype=bf), torch.zeros(10, 2, 64, dtype=bf)
    off, idx = torch.zeros(3, dtype=torch.int32), torch.zeros(10, dtype=torch.int32)
    for bad in (dict(k_cache=k.half()), dict(v_cache=k[:5]), dict(k_cache=k.float(), v_cache=k.float()),
                dict(q=q.transpose(1, 2)), dict(qo_indptr=off[:2]), dict(o=torch.zeros(4, 8, 64)),
                dict(o=torch.zeros(3, 8, 64, dtype=bf))):
        kw = dict(q=q, k_cache=k, v_cache=k, qo_indptr=off, kv_indptr=off, kv_indices=idx)
        kw.update(bad)
        with pytest.raises(L.DFTError):
            K.chunk_attention(**kw)
    with pytest.raises(L.DFTError):
        K.kv_append(q[:, :2], q[:, :2], k, k.half(), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(L.DFTError):
        K.kv_append(q[:, :2], q[:, :2], k, k, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(L.DFTError):
        K.kv_commit(k, k, off, idx, torch.zeros(2, 4, dtype=torch.int64), torch.zeros(3, dtype=torch.int64), 4)
    z, t = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 4, dtype=torch.int32)
    h, f, n = torch.zeros(2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for bad in (dict(fresh=z[:1]), dict(block_table=t.long()), dict(held=h[:1]), dict(tokens=None), dict(n_free=h),
                dict(rows=z[:1]), dict(cached=torch.zeros(3, dtype=torch.int64),
                                       fresh=torch.zeros(3, dtype=torch.int64))):
        kw = dict(cached=z, fresh=z, block_table=t, held=h, free_pages=f, n_free=n, page_size=4, tokens=1)
        kw.update(bad)
        with pytest.raises(L.DFTError):
            K.page_plan(**kw)


def test_oracle_plan_by_hand():
    table, held, stack = np.full((3, 4), -1), np.zeros(3, int), [0, 1, 2, 3, 4]
    got = OP.page_plan([0, 0], [5, 2], [2, 0], table, held, stack, 4)
    assert stack == [0, 1] and table[2].tolist() == [4, 3, -1, -1] and table[0][0] == 2
    assert got == ([0, 5, 7], [0, 5, 7], [16, 17, 18, 19, 12, 8, 9], [16, 17, 18, 19, 12, 8, 9], [0, 1, 2, 3, 4, 0, 1])
    # row 2 shrinks to one page, row 0 takes it back off the stack's top
    got = OP.page_plan([3, 2], [0, 3], [2, 0], table, held, stack, 4)
    assert stack == [0, 1] and table[0].tolist() == [2, 3, -1, -1] and held.tolist() == [2, 0, 1]
    assert got[3] == [10, 11, 12] and got[4] == [2, 3, 4]
    assert OP.page_plan([3, 5], [40, 0], [2, 0], table, held, stack, 4) is None


# rows of 64 elements, two heads, ten slots
OVERLAPS = [dict(kv_st=0), dict(kv_sh=0), dict(kv_st=64, kv_sh=64), dict(kv_st=120, kv_sh=64), dict(kv_sh=32),
            dict(kv_st=-128), dict(kv_sh=-64), dict(kv_st=64, kv_sh=632)]


@pytest.mark.parametrize("kw", OVERLAPS)
def test_append_refuses_caches_whose_rows_overlap(lib, kw):
    assert lib.dft_kv_append(ctypes.byref(_append(**kw)), None, None) == L.DFT_ERR_INVALID


@pytest.mark.parametrize("kw", OVERLAPS + [dict(kv_sl=0), dict(kv_sl=64), dict(kv_sl=1272), dict(kv_sl=-1280)])
def test_commit_refuses_caches_whose_rows_overlap(lib, kw):
    assert lib.dft_kv_commit(ctypes.byref(_commit(L=3, **kw)), None, None) == L.DFT_ERR_INVALID


@pytest.mark.parametrize("kw", [dict(o_st=0), dict(o_sh=0), dict(o_st=64), dict(o_st=504), dict(o_sh=56),
                                dict(o_st=-512), dict(q_st=0), dict(q_sh=0), dict(q_st=-512), dict(n_slots=0),
                                dict(kv_st=56), dict(kv_sh=56), dict(kv_sh=-64)])
def test_attention_refuses_strides_that_name_no_rows(lib, kw):
    a = _attn(**kw)
    assert lib.dft_chunk_attn_workspace_bytes(ctypes.byref(a)) == -1
    assert lib.dft_chunk_attn(ctypes.byref(a), FAKE, None, None) == L.DFT_ERR_INVALID


@pytest.mark.parametrize("kw", [dict(), dict(o_st=64, o_sh=256), dict(T=1, o_st=0, q_st=0), dict(kv_st=64, kv_sh=640),
                                dict(kv_st=256), dict(n_slots=1, kv_st=64, kv_sh=64), dict(q_st=64, q_sh=64),
                                dict(Hq=1, Hkv=1, q_sh=0, o_sh=0, kv_sh=0)])
def test_attention_takes_these_layouts(lib, kw):
    assert lib.dft_chunk_attn_workspace_bytes(ctypes.byref(_attn(**kw))) > 0


def test_wide_offsets_and_slots_do_not_wrap():
    wide = torch.tensor([0, 7, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 7, 2 ** 62, -1, -2 ** 32, -2 ** 40 + 3])
    assert K._offsets(wide).tolist() == [0, 7, 2 ** 31 - 1] + [-1] * 7
    assert K._slots(wide).tolist() == [0, 7] + [2 ** 31 - 1] * 5 + [-1] * 3
    for f in (K._offsets, K._slots):
        same = torch.tensor([3, -5], dtype=torch.int32)
        assert f(same) is same and f(wide).dtype is f(wide[::2]).dtype is torch.int32
        assert f(torch.tensor([3, 4], dtype=torch.int16)).tolist() == [3, 4]


def test_attention_refuses_scales_that_overflow_with_log2_e(lib):
    for scale, rc in ((2.36e38, 1), (2.9e38, 1), (3.4e38, 1), (2.35e38, 0), (1e-38, 0)):
        a = _attn(sm_scale=scale)
        assert (lib.dft_chunk_attn_workspace_bytes(ctypes.byref(a)) == -1) == (rc == 1), scale
