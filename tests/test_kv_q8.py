"""The 8-bit KV cache and its operators on the CPU: the 64-bit oracle's own rules, the C descriptors' layout, and every
refusal of the C entry points (host checks: no launch, so addresses only need to look right)."""

import ctypes as C
import math
import subprocess

import pytest
import torch

from conftest import REPO
from oracle import kv_q8 as ref

BAD, RANGE = 1, 2


def test_rounding_matches_torch_e4m3():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(4000, generator=g) * 100, torch.randn(4000, generator=g) * 0.01,
                   torch.arange(-448, 449, dtype=torch.float32), torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x.clamp(-448, 448)
    assert torch.equal(ref.e4m3(x.double()), x.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.5, 1), (224.0, -1), (225.0, 0), (1.0, -8), (1.75, -8), (1.7578125, -7),
                                    (0.0, -100), (2.0 ** -120, -100), (3.0e38, 120)])
def test_exponent_is_the_least_power_of_two(amax, e):
    assert int(ref.exponent(torch.tensor([amax, -amax / 3, 0.0]))) == e


def test_stored_values_are_bf16_and_idempotent():
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)) * torch.logspace(-20, 20, 50)[:, None]
    y = ref.stored(x)
    assert torch.equal(y.to(torch.bfloat16).double(), y)
    assert torch.equal(ref.stored(y), y)
    # half a step of four significant bits, or half the least step
    step = torch.ldexp(torch.ones(50, dtype=torch.float64), ref.exponent(x) - 10)[:, None]
    assert ((y - x.double()).abs() <= torch.maximum(x.double().abs() * 2 ** -4, step)).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_element_order_is_a_permutation(hd):
    for f in (ref.k_offset, ref.v_offset):
        assert sorted(f(s, d, hd) for s in range(128) for d in range(hd)) == list(range(128 * hd))
    assert sorted(ref.x_offset(s) for s in range(192)) == list(range(192))


def test_header_offsets_agree_with_the_oracle():
    """The formulas documented at SsdKvQ8."""
    for hd in (64, 128):
        for s in range(0, 256, 7):
            for d in range(0, hd, 5):
                assert ref.k_offset(s, d, hd) == ((s // 16) * (hd // 64) + d // 64) * 1024 + (((d // 16) % 4) * 16 + s % 16) * 16 + d % 16
                assert ref.v_offset(s, d, hd) == ((s // 64) * (hd // 16) + d // 16) * 1024 + (((s // 4) % 4) * 16 + d % 16) * 16 + (
                    (s // 32) % 2) * 8 + ((s // 16) % 2) * 4 + s % 4
            assert ref.x_offset(s) == (s // 64) * 64 + ((s // 4) % 4) * 16 + ((s // 16) % 4) * 4 + s % 4


def test_descriptors_have_the_c_layout(tmp_path):
    from ssd import _lib

    structs = {n: getattr(_lib, n) for n in ("SsdKvQ8", "SsdRope")}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{REPO}/include/ssd_mi355x.h"', "int main(void) {"]
    for name, T in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, *_ in T._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, T in structs.items():
        assert int(got[name]) == C.sizeof(T)
        for f, *_ in T._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(T, f).offset, f


# ------------------------------------------------------------------------------------------------- tables
def test_rope_tables_default_and_linear():
    from ssd.models.llama import rope_tables_f32

    cos, sin = rope_tables_f32(5000, 64, 10000.0, "cpu")
    for p, i in ((0, 0), (1, 31), (4999, 0), (4321, 7)):
        a = p * 10000.0 ** (-2 * i / 64)
        assert abs(float(cos[p, i]) - math.cos(a)) < 1e-7 and abs(float(sin[p, i]) - math.sin(a)) < 1e-7
    c4, _ = rope_tables_f32(4000, 64, 10000.0, "cpu", {"rope_type": "linear", "factor": 4.0})
    assert torch.allclose(c4[::4], cos[:1000], atol=1e-6)


def test_rope_tables_llama3_matches_the_bf16_tables():
    from ssd.models.llama import rope_tables, rope_tables_f32

    s = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
    cos, sin = rope_tables_f32(600, 128, 500000.0, "cpu", s)
    cb, sb = rope_tables(600, 128, 500000.0, "cpu", (8.0, 1.0, 4.0, 8192))
    # bf16 tables: half a step of 2^-8, and the fp32 angle's own error (position 600: below 2^-14)
    assert (cos - cb.float()).abs().max() <= 2 ** -9 + 2 ** -13 and (sin - sb.float()).abs().max() <= 2 ** -9 + 2 ** -13


def test_rope_tables_yarn_ends_and_refusals():
    from ssd.models.llama import rope_tables_f32

    s = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=8192)
    cos, sin = rope_tables_f32(16, 128, 500000.0, "cpu", s)
    gain = 0.1 * math.log(4.0) + 1.0
    last = 500000.0 ** (-126 / 128) / 4.0  # the slowest dim is interpolated, the fastest kept
    assert abs(float(sin[3, 0]) - gain * math.sin(3.0)) < 1e-6 and abs(float(sin[3, 63]) - gain * math.sin(3 * last)) < 1e-9
    assert torch.allclose(cos[0], torch.full((64,), gain))
    with pytest.raises(ValueError, match="rope_type"):
        rope_tables_f32(16, 128, 1e4, "cpu", {"rope_type": "dynamic"})
    with pytest.raises(ValueError, match="rot_dim"):
        rope_tables_f32(16, 63, 1e4, "cpu")


# ------------------------------------------------------------------------------------------------- refusals
A = 1 << 20  # an aligned address that is never read


def _cache(**kw):
    from ssd import _lib

    f = dict(k=A, v=A, k_exp=A, v_exp=A, n_seq=2, kv_heads=2, head_dim=128, max_len=128)
    f.update(kw)
    return _lib.SsdKvQ8(*(f[n] for n, *_ in _lib.SsdKvQ8._fields_))


def _rope(**kw):
    from ssd import _lib

    f = dict(cos=A, sin=A, rows=10, rot_dim=64, interleaved=0)
    f.update(kw)
    return _lib.SsdRope(*(f[n] for n, *_ in _lib.SsdRope._fields_))


def _refused(name, args, code, text):
    from ssd import _lib

    lib = _lib.load()
    assert getattr(lib, name)(*args) == code, (name, lib.ssd_last_error())
    assert text in lib.ssd_last_error().decode(), lib.ssd_last_error()


BAD_CACHES = [(dict(k=None), "null"), (dict(v_exp=None), "null"), (dict(head_dim=96), "head_dim"), (dict(head_dim=32), "head_dim"),
              (dict(n_seq=0), "sequences"), (dict(kv_heads=0), "kv heads"), (dict(max_len=100), "max_len"), (dict(max_len=0), "max_len"),
              (dict(max_len=2 ** 30 + 64), "max_len"), (dict(v=A + 8), "aligned")]


def _write(cache=None, **kw):
    f = dict(k=A, ldk=256, v=A, ldv=256, M=3, seq=A, slot=A, rope=None, pos=None, q=None, ldq=0, heads=0, q_out=None, ldo=0)
    f.update(kw)
    f["rope"] = f["rope"] and C.byref(f["rope"])
    return [C.byref(cache or _cache()), *f.values(), None]


@pytest.mark.parametrize("kw,text", BAD_CACHES)
def test_bad_caches_are_refused(kw, text):
    c = _cache(**kw)
    _refused("ssd_kv_q8_write_bf16", _write(c), BAD, text)
    _refused("ssd_kv_q8_read_bf16", [C.byref(c), 1, A, A, A, 256, A, 256, None], BAD, text)
    _refused("ssd_kv_q8_compact", [C.byref(c), 1, A, A, A, 4, None], BAD, text)
    _refused("ssd_tree_attention_q8", [C.byref(c), A, 256, 1, 2, A, A, A, A, 1, 64, 64, 1.0, A, 1 << 20, A, 256, None], BAD, text)


def test_launches_beyond_the_grid_are_refused():
    c = _cache(n_seq=1 << 22, kv_heads=8)
    _refused("ssd_kv_q8_compact", [C.byref(c), 1, A, A, A, 4, None], RANGE, "too large")
    _refused("ssd_kv_q8_write_bf16", _write(_cache(kv_heads=1024), k=A, ldk=1 << 17, ldv=1 << 17, M=1 << 20), RANGE, "too many rows")
    c = _cache(kv_heads=1024)
    _refused("ssd_kv_q8_read_bf16", [C.byref(c), 1 << 20, A, A, A, 1 << 17, A, 1 << 17, None], RANGE, "too many rows")
    args = [C.byref(_cache(n_seq=1 << 20, kv_heads=1)), A, 1024, 1 << 24, 8, A, A, A, A, 64, 128, 64, 1.0, A, 1 << 40, A, 1024, None]
    _refused("ssd_tree_attention_q8", args, RANGE, "workgroups")
    _refused("ssd_kv_q8_compact", [C.byref(_cache(n_seq=1 << 20, kv_heads=1 << 12)), 1, A, A, A, 4, None], RANGE, "sequences")
    args = [A, 1 << 20, 1 << 19, A, 1 << 20, 1 << 19, 1 << 19, 1 << 20, 1, A, None, A, A, A, 1 << 40, A, A, None]
    _refused("ssd_verify_chain", args, RANGE, "sequences")


def test_null_cache_is_refused():
    _refused("ssd_kv_q8_compact", [None, 1, A, A, A, 4, None], BAD, "null cache")


@pytest.mark.parametrize("kw,text", [
    (dict(k=None), "null"), (dict(slot=None), "null"), (dict(M=-1), "M=-1"), (dict(k=A + 2), "aligned"), (dict(ldv=248), "strides"),
    (dict(ldk=260), "strides"), (dict(rope=True), "null rotary"), (dict(q=A, heads=4, ldq=512), "q/q_out"),
    (dict(q=A, heads=4, ldq=500, q_out=A, ldo=512), "q/q_out"), (dict(q=A, heads=0, ldq=512, q_out=A, ldo=512), "q/q_out")])
def test_write_refusals(kw, text):
    if kw.get("rope"):
        kw = dict(kw, rope=_rope())  # tables without positions
    _refused("ssd_kv_q8_write_bf16", _write(**kw), BAD, text)


@pytest.mark.parametrize("kw", [dict(rot_dim=8), dict(rot_dim=72), dict(rot_dim=144), dict(rot_dim=0)])
def test_rot_dim_refusals(kw):
    _refused("ssd_kv_q8_write_bf16", _write(rope=_rope(**kw), pos=A), BAD, "rot_dim")
    _refused("ssd_rope_bf16", [C.byref(_rope(**kw)), A, A, 256, 2, 2, 128, A, 256, None], BAD, "rot_dim")


def test_rope_refusals():
    r = C.byref(_rope())
    _refused("ssd_rope_bf16", [None, A, A, 256, 2, 2, 128, A, 256, None], BAD, "null")
    _refused("ssd_rope_bf16", [r, None, A, 256, 2, 2, 128, A, 256, None], BAD, "null")
    _refused("ssd_rope_bf16", [r, A, A, 256, 2, 2, 96, A, 256, None], BAD, "head_dim")
    _refused("ssd_rope_bf16", [r, A, A, 256, 2, 0, 128, A, 256, None], BAD, "heads")
    _refused("ssd_rope_bf16", [r, A, A, 248, 2, 2, 128, A, 256, None], BAD, "strides")


def test_read_and_compact_refusals():
    c = C.byref(_cache())
    _refused("ssd_kv_q8_read_bf16", [c, 1, None, A, A, 256, A, 256, None], BAD, "null")
    _refused("ssd_kv_q8_read_bf16", [c, -1, A, A, A, 256, A, 256, None], BAD, "M=-1")
    _refused("ssd_kv_q8_read_bf16", [c, 1, A, A, A, 128, A, 256, None], BAD, "strides")
    _refused("ssd_kv_q8_compact", [c, 0, A, A, A, 4, None], BAD, "layers")
    _refused("ssd_kv_q8_compact", [c, 1, A, None, A, 4, None], BAD, "null")
    _refused("ssd_kv_q8_compact", [c, 1, A, A, A, 65, None], RANGE, "n_max")


@pytest.mark.parametrize("at,value,code,text", [
    (1, None, BAD, "null"), (13, None, BAD, "null"), (3, -1, BAD, "M=-1"), (4, 3, BAD, "heads"), (4, 0, BAD, "heads"), (9, 0, RANGE, "rows"),
    (9, 65, RANGE, "rows"), (10, 0, BAD, "l_max"), (10, 129, BAD, "l_max"), (11, 32, BAD, "span"), (11, 96, BAD, "span"), (12, -1.0, BAD, "scale"), (12, 0.0, BAD, "scale"),
    (12, float("nan"), BAD, "scale"), (12, float("inf"), BAD, "scale"), (2, 508, BAD, "strides"),
    (1, A + 8, BAD, "aligned"), (16, 504, BAD, "strides"), (14, 100, BAD, "workspace"), (13, A + 4, BAD, "workspace")])
def test_attention_refusals(at, value, code, text):
    args = [C.byref(_cache()), A, 512, 5, 4, A, A, A, A, 5, 128, 64, 1.0, A, 5 * 4 * 2 * 130, A, 512, None]
    args[at] = value
    _refused("ssd_tree_attention_q8", args, code, text)


@pytest.mark.parametrize("at,value,code,text", [
    (0, None, BAD, "null"), (3, None, BAD, "null"), (9, None, BAD, "null"), (11, None, BAD, "null"), (12, None, BAD, "null"), (15, None, BAD, "null"),
    (6, 0, BAD, "V=0"), (6, (1 << 24) + 1, RANGE, "columns"), (7, -1, BAD, "n_seq"), (8, -1, BAD, "k_max"), (8, 65, RANGE, "drafted"),
    (2, 99, BAD, "strides"), (5, 99, BAD, "strides"), (13, A + 4, BAD, "aligned"), (14, 95, BAD, "workspace")])
def test_verify_chain_refusals(at, value, code, text):
    args = [A, 400, 100, A, 300, 100, 100, 3, 3, A, None, A, A, A, 96, A, A, None]
    args[at] = value
    _refused("ssd_verify_chain", args, code, text)


def test_workspace_sizes():
    from ssd import _lib

    lib = _lib.load()
    assert lib.ssd_attn_q8_ws_floats(3, 8, 128, 600, 128) == 3 * 8 * 2 * 130
    assert lib.ssd_attn_q8_ws_floats(3, 8, 128, 300, 100) == -1 and lib.ssd_attn_q8_ws_floats(3, 8, 128, 0, 64) == -1
    assert lib.ssd_attn_q8_ws_floats(64, 64, 128, 1 << 20, 64) == 64 * 64 * (1 << 12) * 130  # past 32 bits
    assert lib.ssd_verify_chain_ws_bytes(3, 4097) == 3 * 3 * 16 and lib.ssd_verify_chain_ws_bytes(3, 0) == -1


def test_python_refusals_without_a_gpu():
    from ssd.engine.kv_cache import KVCacheQ8
    from ssd import ops

    with pytest.raises(ValueError, match="head_dim"):
        KVCacheQ8(1, 64, 2, 96, "cpu")
    with pytest.raises(ValueError, match="span"):
        KVCacheQ8(1, 64, 2, 64, "cpu", span=100)
    with pytest.raises(ValueError, match="positive"):
        KVCacheQ8(1, 0, 2, 64, "cpu")
    t = torch.zeros(4, 8)
    for cos, sin in ((t, t[:, :4]), (t.double(), t.double()), (t[:, ::2], t[:, ::2]), (t[0], t[0])):
        with pytest.raises(ValueError, match="rotary tables"):
            ops.RopeTables(cos, sin)


def test_a_prompt_of_another_shape_is_not_loaded():
    from ssd.engine.kv_cache import KVCache, KVCacheQ8

    cache = KVCacheQ8(1, 256, 2, 64, "cpu")
    for other in (KVCache(1, 256, 4, 64, "cpu"), KVCache(1, 256, 2, 128, "cpu"), KVCache(1, 100, 2, 64, "cpu")):
        with pytest.raises(ValueError, match="slots of 2 heads of 64 from a cache"):
            cache.load(0, other, 120)


def test_a_span_beyond_the_kernels_is_refused():
    from ssd.engine.kv_cache import KVCacheQ8

    with pytest.raises(ValueError, match="span"):
        KVCacheQ8(1, 64, 2, 64, "cpu", span=(1 << 20) + 64)


def test_descriptors_keep_their_arrays_and_their_layers(monkeypatch):
    import gc
    import weakref

    from ssd import ops
    from ssd.engine.kv_cache import KVCacheQ8

    cache = KVCacheQ8(3, 64, 2, 64, "cpu")
    seen, first, second = weakref.ref(cache.k), cache.k.data_ptr(), cache.layer(1)
    del cache
    gc.collect()
    assert seen() is not None and second.k == first + seen()[0].numel()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    start = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="3 layers of a cache that holds 2"):
        ops.kv_q8_compact(second, 3, start, start[None], start, 1)


def test_made_outputs_have_the_rows_that_are_written(monkeypatch):
    from ssd import ops
    from ssd.engine.kv_cache import KVCacheQ8

    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops._lib, "call", lambda *a: 0)
    cache = KVCacheQ8(1, 64, 2, 64, "cpu")
    i = torch.zeros(8, dtype=torch.int32)
    q, k = torch.zeros(5, 256, dtype=torch.bfloat16), torch.zeros(3, 128, dtype=torch.bfloat16)
    assert cache.write(0, k, k, i, i, q=q).shape == (3, 256)
    out = ops.tree_attention_q8(cache.layer(0), q, 3, 4, i, i, i, torch.zeros(8, 32, dtype=torch.int32), 1, 64, 64)
    assert out.shape == (3, 256)


def test_a_dropped_cache_frees_its_arrays():
    """With no descriptor held, after a held one goes, and after the descriptors were used by calls."""
    import gc
    import weakref

    from ssd.engine.kv_cache import KVCacheQ8

    def arrays(cache):
        return [weakref.ref(t) for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)]

    cache = KVCacheQ8(3, 64, 2, 64, "cpu")
    seen = arrays(cache)
    del cache
    gc.collect()
    assert not any(r() is not None for r in seen)

    cache = KVCacheQ8(3, 64, 2, 64, "cpu")
    seen, held = arrays(cache), cache.layer(1)
    del cache
    gc.collect()
    assert all(r() is not None for r in seen)
    del held
    gc.collect()
    assert not any(r() is not None for r in seen)


def test_calls_keep_no_cache(monkeypatch):
    import gc
    import weakref

    from ssd import ops
    from ssd.engine.kv_cache import KVCacheQ8

    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops._lib, "call", lambda name, *args: C.POINTER(ops._lib.SsdKvQ8).from_param(args[0]) and 0)
    cache = KVCacheQ8(2, 64, 2, 64, "cpu")
    seen = weakref.ref(cache.k)
    i = torch.zeros(8, dtype=torch.int32)
    k, q = torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, 256, dtype=torch.bfloat16)
    cache.write(0, k, k, i, i)
    cache.read(1, i, i)
    cache.attend(0, q, i, i, i, torch.zeros(8, 32, dtype=torch.int32), 3, 64)
    cache.compact_device(i, i[None], i)
    del cache
    gc.collect()
    assert seen() is None


def _calls_without_a_gpu(monkeypatch):
    from ssd import ops

    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops._lib, "call", lambda *a: 0)


@pytest.mark.parametrize("shape", [(3, 64), (6, 16), (3, 33), (96, 1), (1, 96), (2, 32)])
def test_ancestor_tables_of_another_width_are_refused(monkeypatch, shape):
    """Rows of a table that is not 32 wide would be read as rows of 32."""
    from ssd.engine.kv_cache import KVCacheQ8

    _calls_without_a_gpu(monkeypatch)
    cache = KVCacheQ8(1, 64, 2, 64, "cpu")
    i, q = torch.zeros(8, dtype=torch.int32), torch.zeros(3, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="anc"):
        cache.attend(0, q, i, i, i, torch.zeros(shape, dtype=torch.int32), 3, 64)


@pytest.mark.parametrize("shape", [(3, 32), (5, 32), (96,), (1, 3, 32)])
def test_ancestor_tables_of_rows_of_32_are_taken(monkeypatch, shape):
    from ssd.engine.kv_cache import KVCacheQ8

    _calls_without_a_gpu(monkeypatch)
    cache = KVCacheQ8(1, 64, 2, 64, "cpu")
    i, q = torch.zeros(8, dtype=torch.int32), torch.zeros(3, 256, dtype=torch.bfloat16)
    assert cache.attend(0, q, i, i, i, torch.zeros(shape, dtype=torch.int32), 3, 64).shape == (3, 256)


def test_moves_of_another_width_are_refused(monkeypatch):
    """Rows of `src` that are not n_max wide would be read as rows of n_max."""
    from ssd import ops
    from ssd.engine.kv_cache import KVCacheQ8

    _calls_without_a_gpu(monkeypatch)
    cache = KVCacheQ8(2, 64, 2, 64, "cpu", sequences=3)
    i = torch.zeros(3, dtype=torch.int32)
    for shape in ((3, 9), (4, 6), (3, 4), (15, 1), (1, 15)):
        with pytest.raises(ValueError, match="src"):
            ops.kv_q8_compact(cache.layer(0), 2, i, torch.zeros(shape, dtype=torch.int32), i, 5)
    for shape in ((3, 5), (4, 5), (15,)):
        ops.kv_q8_compact(cache.layer(0), 2, i, torch.zeros(shape, dtype=torch.int32), i, 5)


def test_no_moves_take_any_table(monkeypatch):
    from ssd import ops
    from ssd.engine.kv_cache import KVCacheQ8

    _calls_without_a_gpu(monkeypatch)
    cache = KVCacheQ8(1, 64, 2, 64, "cpu", sequences=3)
    i = torch.zeros(3, dtype=torch.int32)
    ops.kv_q8_compact(cache.layer(0), 1, i, torch.zeros(3, 9, dtype=torch.int32), i, 0)
    cache.compact_device(i, torch.zeros(3, 0, dtype=torch.int32), i)


@pytest.mark.parametrize("extra,gain", [
    ({}, 0.1 * math.log(40) + 1), (dict(mscale=1.0, mscale_all_dim=1.0), 1.0),
    (dict(mscale=0.707, mscale_all_dim=1.0), (0.0707 * math.log(40) + 1) / (0.1 * math.log(40) + 1)),
    (dict(mscale=1.5), 0.1 * math.log(40) + 1), (dict(mscale=1.0, mscale_all_dim=0), 0.1 * math.log(40) + 1),
    (dict(attention_factor=0.75, mscale=0.707, mscale_all_dim=1.0), 0.75), (dict(factor=1.0), 1.0),
    (dict(factor=0.5, mscale=2.0, mscale_all_dim=1.0), 1.0), (dict(attention_factor=None, mscale=None), 0.1 * math.log(40) + 1)])
def test_rope_tables_yarn_factor_on_cos_and_sin(extra, gain):
    """Position 0: cos is the factor. attention_factor as given; else the ratio of the two scales' 0.1 s ln(factor) + 1 where
    both are given (and not 0); else 0.1 ln(factor) + 1; a factor of at most 1 scales by 1."""
    from ssd.models.llama import rope_tables_f32

    s = dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096)
    cos, _ = rope_tables_f32(2, 64, 10000.0, "cpu", {**s, **extra})
    assert float((cos[0] - gain).abs().max()) <= gain * 2 ** -24  # one rounding to fp32


@pytest.mark.parametrize("truncate", [None, True, False])
@pytest.mark.parametrize("rot,theta,context,fast,slow", [(128, 500000.0, 8192, 32.0, 1.0), (64, 10000.0, 4096, 32.0, 1.0),
                                                         (64, 150000.0, 4096, 32.0, 1.0), (32, 1e4, 16384, 8.0, 2.0)])
def test_rope_tables_yarn_inside_the_ramp(rot, theta, context, fast, slow, truncate):
    """Every dim's frequency against the definition, dim by dim: a dim that turns `fast` times or more in the original context
    stays, one that turns `slow` times or less is divided by the factor, between them linear in the dim's number; the ends of the ramp are
    whole dims (rounded outwards) unless truncate is False."""
    from ssd.models.llama import rope_tables_f32

    f = 4.0
    s = dict(rope_type="yarn", factor=f, original_max_position_embeddings=context, beta_fast=fast, beta_slow=slow, attention_factor=1.0)
    if truncate is not None:
        s["truncate"] = truncate
    _, sin = rope_tables_f32(2, rot, theta, "cpu", s)
    # theta^(2 d / rot) = context / (2 pi turns) at dim d
    first, last = (math.log(context / (2 * math.pi * turns), theta) * rot / 2 for turns in (fast, slow))
    if truncate is not False:
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rot - 1)
    inside = 0
    for d in range(rot // 2):
        t = min(max((d - first) / (last - first), 0.0), 1.0)
        inside += 0 < t < 1
        w = theta ** (-2 * d / rot)
        want = math.sin(w * (1 - t) + w / f * t)  # position 1
        assert abs(float(sin[1, d]) - want) <= abs(want) * (2 ** -24 + 2 ** -40), d  # one rounding; the doubles' own far below
    assert inside >= 2  # the shortest ramp, 10.05 to 12.46, holds dims 11 and 12


def test_a_prompt_may_fill_the_capacity(monkeypatch):
    """Every slot of the capacity exists for write, read, attend and compaction, and for load alike."""
    from ssd.engine.kv_cache import KVCache, KVCacheQ8

    _calls_without_a_gpu(monkeypatch)
    cache, full = KVCacheQ8(1, 200, 2, 64, "cpu"), KVCache(1, 300, 2, 64, "cpu")
    assert cache.capacity == 256
    written = []
    monkeypatch.setattr(cache, "write", lambda i, k, v, seq, slot: written.append(slot.tolist()))
    cache.load(0, full, 256, start=190)
    assert written == [list(range(190, 256))]
    for args in ((257,), (10, 0, 11), (10, 1), (10, 0, -1)):
        with pytest.raises(ValueError, match="load"):
            cache.load(0, full, *args)
