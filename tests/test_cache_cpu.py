"""CPU tests of the 4-bit key/value cache: refusals at the C ABI and in the binding, the layout of
the structs, and the oracle's format."""
import ctypes
import math
import os

import pytest
import torch

from oracle import cache_oracle as oracle
from w4a16_opt import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000      # an aligned address that is never read: every call here is refused before a launch


def cache(**kw):
    c = dict(data=P, num_pages=4, page_size=64, kv_heads=2, head_dim=128, group_size=128)
    c.update(kw)
    return capi.Cache(**c)


def rotary(**kw):
    r = dict(q=P, q_out=P, q_token_stride=1024, q_head_stride=128, positions=P, positions_axis_stride=0, cos_sin=P,
             max_pos=100, q_heads=8, axes=1, rotary_dim=128, interleaved=0)
    sections = kw.pop("sections", (0, 0, 0))
    r.update(kw)
    out = capi.Rotary(**r)
    out.sections = (ctypes.c_int32 * 3)(*sections)
    return out


def append(c=None, k=P, v=P, strides=(256, 128, 256, 128), dtype=0, slots=P, tokens=5, rot=None):
    lib = capi.load()
    c = cache() if c is None else c
    st = lib.w4a16_cache_append(ctypes.byref(c), k, v, *strides, dtype, slots, tokens,
                                ctypes.byref(rot) if rot is not None else None, None)
    return st, capi.last_error(lib)


def args(**kw):
    a = dict(q=P, out=P, lse=None, q_token_stride=1024, q_head_stride=128, q_tokens=3, page_table=P, page_table_stride=4,
             seq_lens=P, cu_q=None, scale=0.1, dtype=0, q_heads=8, batch=3, table_pages=4, max_q=1, causal=1, window=0)
    a.update(kw)
    return capi.CacheAttentionArgs(**a)


def attention(c=None, **kw):
    lib = capi.load()
    c = cache() if c is None else c
    st = lib.w4a16_cache_attention(ctypes.byref(c), ctypes.byref(args(**kw)), None, 0, None)
    return st, capi.last_error(lib)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(head_dim=96), 19, "unsupported head_dim 96"),
    (dict(head_dim=0), 19, "unsupported head_dim"),
    (dict(group_size=32), 10, "unsupported group size 32"),
    (dict(head_dim=64, group_size=128), 10, "at most head_dim"),
    (dict(page_size=48), 19, "unsupported page_size 48"),
    (dict(page_size=-16), 19, "unsupported page_size"),
    (dict(kv_heads=0), 19, "kv_heads"),
    (dict(kv_heads=1025), 19, "kv_heads"),
    (dict(num_pages=0), 19, "num_pages"),
    (dict(num_pages=1 << 31), 19, "num_pages"),
])
def test_caches_that_are_refused(kw, status, msg):
    for st, err in (append(cache(**kw)), attention(cache(**kw))):
        assert st == status and msg in err, (st, err)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=2), 20, "dtype must be 0 (fp16) or 1 (bf16)"),
    (dict(tokens=-1), 4, "fit in int32"),
    (dict(tokens=1 << 30), 4, "fit in int32"),
    (dict(c=cache(data=None)), 1, "non-null"),
    (dict(k=None), 1, "non-null"),
    (dict(slots=None), 1, "non-null"),
    (dict(k=P + 8), 9, "16-byte aligned"),
    (dict(c=cache(data=P + 4)), 9, "16-byte aligned"),
    (dict(strides=(256, 129, 256, 128)), 9, "multiples of 8"),
    (dict(strides=(256, 128, 260, 128)), 9, "multiples of 8"),
    (dict(rot=rotary(rotary_dim=96)), 19, "rotary_dim"),
    (dict(rot=rotary(axes=0)), 19, "1 to 3 axes"),
    (dict(rot=rotary(axes=4)), 19, "1 to 3 axes"),
    (dict(rot=rotary(axes=3, sections=(16, 24, 25))), 19, "add up"),
    (dict(rot=rotary(axes=2, sections=(-1, 65, 0))), 19, "negative"),
    (dict(rot=rotary(max_pos=0)), 19, "at least one position"),
    (dict(rot=rotary(q_heads=0)), 19, "q_heads"),
    (dict(rot=rotary(positions=None)), 1, "non-null"),
    (dict(rot=rotary(q_out=None)), 1, "non-null"),
    (dict(rot=rotary(cos_sin=P + 4)), 9, "aligned"),
    (dict(rot=rotary(q_token_stride=1025)), 9, "multiples of 8"),
])
def test_appends_that_are_refused(kw, status, msg):
    st, err = append(**kw)
    assert st == status and msg in err, (st, err)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=7), 20, "dtype"),
    (dict(q_heads=7), 19, "multiple of kv_heads"),
    (dict(q_heads=0), 19, "multiple of kv_heads"),
    (dict(batch=-1), 19, "batch"),
    (dict(batch=65536), 19, "batch"),
    (dict(table_pages=-1), 19, "table_pages"),
    (dict(table_pages=1 << 26), 4, "table_pages * page_size"),
    (dict(q_tokens=-1), 4, "q_tokens"),
    (dict(q_tokens=1 << 30), 4, "fit in int32"),
    (dict(max_q=4), 19, "max_q"),
    (dict(max_q=-1), 19, "max_q"),
    (dict(max_q=2), 19, "without cu_q"),
    (dict(window=-1), 19, "window"),
    (dict(scale=math.nan), 19, "scale"),
    (dict(q=None), 1, "non-null"),
    (dict(out=None), 1, "non-null"),
    (dict(seq_lens=None), 1, "non-null"),
    (dict(page_table=None), 1, "non-null"),
    (dict(q=P + 2), 9, "16-byte aligned"),
    (dict(q_head_stride=12), 9, "multiples of 8"),
])
def test_attention_that_is_refused(kw, status, msg):
    st, err = attention(**kw)
    assert st == status and msg in err, (st, err)


def test_calls_without_work_need_no_device():
    assert append(tokens=0, k=None, slots=None)[0] == 0
    assert attention(batch=0)[0] == 0
    assert attention(q_tokens=0, max_q=0)[0] == 0
    lib = capi.load()
    assert lib.w4a16_cache_read(ctypes.byref(cache()), None, 0, None, None, 0, None) == 0
    assert lib.w4a16_cache_read(ctypes.byref(cache()), P, 5, P, P + 8, 0, None) == 9
    assert lib.w4a16_cache_read(ctypes.byref(cache()), P, 5, None, P, 0, None) == 1
    assert lib.w4a16_cache_read(ctypes.byref(cache()), P, 5, P, P, 3, None) == 20


def test_null_structs_are_refused():
    lib = capi.load()
    a, c = args(), cache()
    assert lib.w4a16_cache_attention(None, ctypes.byref(a), None, 0, None) == 1
    assert lib.w4a16_cache_attention(ctypes.byref(c), None, None, 0, None) == 1
    assert lib.w4a16_cache_append(None, P, P, 8, 8, 8, 8, 0, P, 1, None, None) == 1
    assert lib.w4a16_cache_page_bytes(64, 128, 128, None) == 1
    assert lib.w4a16_cache_attention_workspace(ctypes.byref(c), ctypes.byref(a), None) == 1


@pytest.mark.parametrize("ps,d,g", [(16, 64, 64), (64, 128, 64), (256, 128, 128)])
def test_page_bytes(ps, d, g):
    n = ctypes.c_uint64()
    assert capi.load().w4a16_cache_page_bytes(ps, d, g, ctypes.byref(n)) == 0
    assert n.value == oracle.block_bytes(ps, d, g) and n.value % 16 == 0


@pytest.mark.skipif(__import__("shutil").which("gcc") is None, reason="needs gcc")
def test_struct_layout_matches_ctypes(tmp_path):
    import subprocess
    structs = {"w4a16_cache": capi.Cache, "w4a16_rotary": capi.Rotary, "w4a16_cache_attention_args": capi.CacheAttentionArgs}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "w4a16.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'    printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'    printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["    return 0;", "}"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src),
                    "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, cls in structs.items():
        assert int(out[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(out[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)


# ------------------------------------------------------------------------------ the binding, on CPU tensors

def test_binding_refuses_cpu_tensors_and_wrong_types():
    import w4a16_opt as w
    data = torch.zeros(2, 1, oracle.block_bytes(16, 64, 64), dtype=torch.uint8)
    c = w.Int4KVCache.wrap(data, 64, 16)
    x, slots = torch.zeros(1, 1, 64, dtype=torch.half), torch.zeros(1, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA"):
        w.cache_append(c, x, x, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        w.cache_read(c, slots)
    with pytest.raises(RuntimeError, match="dtype must be fp16 or bf16"):
        w.cache_read(c, slots, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        w.cache_attention(x, c, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="cu_q needs max_q"):
        w.cache_attention(x, c, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                          cu_q=torch.zeros(2, dtype=torch.int32))
    for bad in (data[:, :, 1:], data.int(), data[0]):
        with pytest.raises(RuntimeError, match="contiguous uint8"):
            w.Int4KVCache.wrap(bad, 64, 16)
    with pytest.raises(RuntimeError, match="unsupported page_size"):
        w.Int4KVCache(2, 1, 64, page_size=20, device="cpu")
    with pytest.raises(RuntimeError, match="unsupported head_dim"):
        w.Int4KVCache(2, 1, 80, group_size=64, device="cpu")


def test_cache_object():
    import w4a16_opt as w
    c = w.Int4KVCache(3, 5, 128, 32, 64, device="cpu")
    assert (c.num_pages, c.kv_heads, c.head_dim, c.page_size, c.group_size) == (3, 5, 128, 32, 64)
    assert c.data.shape == (3, 5, 32 * (128 + 16)) and c.data.dtype == torch.uint8 and not c.data.any()
    assert w.Int4KVCache(1, 1, 64, device="cpu").group_size == 64


# ------------------------------------------------------------------------------ the oracle

@pytest.mark.parametrize("d,g,ps", [(64, 64, 16), (128, 64, 32), (128, 128, 16)])
def test_oracle_blocks_round_trip(d, g, ps):
    gen = torch.Generator().manual_seed(d + g)
    x = torch.randn(2, 7, 2, d, generator=gen).half()
    data = torch.zeros(2, 2, oracle.block_bytes(ps, d, g), dtype=torch.uint8)
    slots = torch.tensor([0, ps + 3, 5, 2 * ps - 1, 1, ps, 9])
    kq, vq = oracle.quantise(x[0], g), oracle.quantise(x[1], g)
    for t, s in enumerate(slots.tolist()):
        for h in range(2):
            oracle.write_block(data[s // ps, h], ps, s % ps, [y[t, h] for y in kq], [y[t, h] for y in vq])
    k, v = oracle.read_slots(data, d, ps, g, slots)
    for got, ref in ((k, x[0]), (v, x[1])):
        rng = ref.double().reshape(7, 2, d // g, g)
        step = ((rng.amax(-1) - rng.amin(-1)) / 15).repeat_interleave(g, -1)
        assert ((got - ref.double()).abs() <= step * 0.505).all()      # half a step, and the scale's rounding


def test_oracle_attention_matches_a_loop():
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 64, generator=gen, dtype=torch.float64) for n, h in ((3, 4), (6, 2), (6, 2)))
    out, lse, spread, _ = oracle.attention(q, k, v, window=2)
    for t in range(3):
        for h in range(4):
            seen = [j for j in range(6) if j <= 3 + t and j > 3 + t - 2]
            s = torch.tensor([float(q[t, h] @ k[j, h // 2]) / 8 for j in seen])
            w = torch.softmax(s.double(), 0)
            want = sum(w[n] * v[j, h // 2] for n, j in enumerate(seen))
            assert (out[t, h] - want).abs().max() < 1e-6
            assert abs(lse[t, h] - torch.logsumexp(s.double(), 0)) < 1e-6
