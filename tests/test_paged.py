"""The paged cache's operators and token log probabilities on the CPU: the 64-bit oracle's own rules, the descriptors' layout, the
page counts, and every refusal of the C entry points (host checks: no launch, so addresses only need to look right)."""

import ctypes as C
import subprocess

import pytest
import torch

from conftest import REPO
from oracle import paged as ref

BAD, RANGE = 1, 2
A = 1 << 20  # an aligned address that is never read


def test_descriptors_have_the_c_layout(tmp_path):
    from ssd import _lib

    structs = {n: getattr(_lib, n) for n in ("SsdPagedKv", "SsdPagedBatch")}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{REPO}/include/ssd_mi355x.h"', "int main(void) {"]
    for name, T in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, *_ in T._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return SSD_PAGE_SLOTS != 64; }"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, T in structs.items():
        assert int(got[name]) == C.sizeof(T)
        for f, *_ in T._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(T, f).offset, f


def test_oracle_attention_is_softmax_and_zeros():
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(3, 4, 8, generator=g), torch.randn(5, 2, 8, generator=g), torch.randn(5, 2, 8, generator=g)
    out, _, w, _ = ref.attention(q, k, v, [-1, 2, 4])
    assert not out[0].any() and torch.allclose(w.sum(-1)[1:], torch.ones(2, 4, dtype=torch.float64))
    s = torch.softmax(k[:3, 1].double() @ q[1, 3].double() / 8 ** 0.5, 0)
    assert torch.allclose(out[1, 3], s @ v[:3, 1].double()) and not w[1, :, 3:].any()


def test_oracle_eviction_rules():
    w = torch.tensor([0.0, 3.0, 1.0, 3.0, float("nan"), 2.0, 0.5, 9.0])
    assert ref.evict(w, 8, 8, 1, 1) == list(range(8)) and ref.evict(w, 3, 4, 1, 1) == [0, 1, 2]
    assert ref.evict(w, 8, 4, 2, 1) == [0, 1, 6, 7]  # of two equal weights the lower slot
    assert ref.evict(w, 8, 5, 0, 0) == [1, 2, 3, 5, 7] and ref.evict(w, 8, 7, 1, 0) == [0, 1, 2, 3, 5, 6, 7]
    assert ref.evict(w, 8, 3, 3, 0) == [5, 6, 7] and ref.evict(w, 8, 2, 0, 2) == [0, 1]


def _kv(**kw):
    from ssd import _lib

    d = dict(k=A, v=A, pages=4, kv_heads=2, head_dim=64) | kw
    return _lib.SsdPagedKv(*(d[n] for n, _ in _lib.SsdPagedKv._fields_))


def _batch(**kw):
    from ssd import _lib

    d = dict(table=A, ld_table=3, table_cols=3, n_seq=2, row_begin=A, lengths=A, rows_max=4) | kw
    return _lib.SsdPagedBatch(*(d[n] for n, _ in _lib.SsdPagedBatch._fields_))


def _refused(name, args, code, text):
    from ssd import _lib

    lib = _lib.load()
    before = lib.ssd_launch_count()
    assert getattr(lib, name)(*args) == code, lib.ssd_last_error()
    assert text in lib.ssd_last_error().decode() and lib.ssd_launch_count() == before


DESCRIPTORS = [(dict(k=None), {}, BAD, "null"), (dict(v=A + 2), {}, BAD, "aligned"), (dict(head_dim=32), {}, BAD, "head_dim"),
               (dict(head_dim=96), {}, BAD, "head_dim"), (dict(pages=0), {}, BAD, "pages"), (dict(kv_heads=0), {}, BAD, "kv_heads"),
               ({}, dict(table=None), BAD, "null"), ({}, dict(lengths=None), BAD, "null"), ({}, dict(n_seq=-1), BAD, "n_seq"),
               ({}, dict(table_cols=0), BAD, "table_cols"), ({}, dict(ld_table=2), BAD, "ld_table"), ({}, dict(rows_max=-1), BAD, "rows_max"),
               ({}, dict(row_begin=None), BAD, "row_begin"), ({}, dict(table_cols=1 << 25, ld_table=1 << 25), RANGE, "2^24")]


@pytest.mark.parametrize("kv,batch,code,text", DESCRIPTORS)
def test_bad_descriptors_are_refused_everywhere(kv, batch, code, text):
    c, b = _kv(**kv), _batch(**batch)
    for name, args in (("ssd_paged_write_bf16", (c, b, A, 128, A, 128, 4, None)), ("ssd_paged_read_bf16", (c, b, 4, A, 128, A, 128, None)),
                       ("ssd_paged_attention_bf16", (c, b, A, 256, 4, 4, 64, 64, 0.1, A, 1 << 20, None, 0, 0, 1.0, A, 256, None)),
                       ("ssd_paged_prompt_bf16", (c, b, A, 256, 4, 4, 64, 0.1, A, 1 << 20, A, 256, None)),
                       ("ssd_paged_evict", (c, 1, 1 << 20, b, _batch(), A, 192, 192, 8, 1, 1, A + 4096, A, None))):
        _refused(name, args, code, text)


ROWS = [(0, None, "null"), (2, None, "null"), (0, A + 8, "aligned"), (1, 120, "strides"), (1, 132, "aligned"), (3, 100, "strides"), (4, -1, "M=-1")]


@pytest.mark.parametrize("at,value,text", ROWS)
def test_bad_rows_are_refused(at, value, text):
    args = [A, 128, A, 128, 4]
    args[at] = value
    _refused("ssd_paged_write_bf16", (_kv(), _batch(), *args, None), BAD, text)
    _refused("ssd_paged_read_bf16", (_kv(), _batch(), args[4], *args[:4], None), BAD, text)


ATTEND = [(dict(q=None), BAD, "null"), (dict(ws=None), BAD, "null"), (dict(out=None), BAD, "null"), (dict(M=-1), BAD, "M=-1"),
          (dict(heads=3), BAD, "heads=3"), (dict(heads=0), BAD, "heads=0"), (dict(l_max=0), BAD, "l_max"), (dict(l_max=193), BAD, "l_max"),
          (dict(span=32), BAD, "span"), (dict(span=100), BAD, "span"), (dict(span=8192), BAD, "span"), (dict(scale=0.0), BAD, "scale"),
          (dict(scale=float("nan")), BAD, "scale"), (dict(q=A + 8), BAD, "aligned"), (dict(ldq=252), BAD, "aligned"),
          (dict(ldo=248), BAD, "strides"), (dict(ws_floats=10), BAD, "workspace"), (dict(ws=A + 4), BAD, "workspace"),
          (dict(weights=A, ldw=100, ldw_seq=1000), BAD, "weights"), (dict(weights=A, ldw=192, ldw_seq=192), BAD, "weights"),
          (dict(weights=A, ldw=192, ldw_seq=384, decay=-0.1), BAD, "decay"), (dict(weights=A, ldw=192, ldw_seq=384, decay=1.5), BAD, "decay"),
          (dict(weights=A, ldw=192, ldw_seq=384, decay=float("nan")), BAD, "decay")]


@pytest.mark.parametrize("kw,code,text", ATTEND)
def test_bad_attention_is_refused(kw, code, text):
    d = dict(q=A, ldq=256, M=4, heads=4, l_max=192, span=64, scale=0.1, ws=A, ws_floats=1 << 20, weights=None, ldw_seq=0, ldw=0, decay=1.0,
             out=A, ldo=256) | kw
    _refused("ssd_paged_attention_bf16", (_kv(), _batch(), *d.values(), None), code, text)
    if not {"ws", "ws_floats", "span", "weights"} & set(kw):
        args = [d[n] for n in ("q", "ldq", "M", "heads", "l_max", "scale", "ws", "ws_floats", "out", "ldo")]
        _refused("ssd_paged_prompt_bf16", (_kv(), _batch(), *args, None), code, text)


def test_grids_beyond_a_launch_are_refused():
    big = _batch(n_seq=1 << 24, rows_max=1000)
    _refused("ssd_paged_write_bf16", (_kv(), big, A, 128, A, 128, 1 << 20, None), RANGE, "workgroups")
    _refused("ssd_paged_attention_bf16", (_kv(), big, A, 256, 1 << 20, 4, 64, 64, 0.1, A, 1 << 60, None, 0, 0, 1.0, A, 256, None), RANGE, "workgroups")
    _refused("ssd_paged_prompt_bf16", (_kv(), big, A, 256, 1 << 20, 4, 64, 0.1, A, 1 << 60, A, 256, None), RANGE, "workgroups")
    _refused("ssd_paged_prompt_bf16", (_kv(), _batch(), A, 256, 1 << 29, 4, 64, 0.1, A, 1 << 60, A, 256, None), RANGE, "rows")
    _refused("ssd_paged_evict", (_kv(), 64, 1 << 20, big, _batch(n_seq=1 << 24), A, 192, 192, 8, 1, 1, A + 4096, A, None), RANGE, "workgroups")


EVICT = [(dict(weights=None), "null"), (dict(out_weights=None), "null"), (dict(kept=None), "null"), (dict(layers=0), "layers"),
         (dict(layer_elems=100), "layer_elems"), (dict(cap=0), "cap"), (dict(ldw=100), "ldw"), (dict(keep=0), "keep"), (dict(recent=-1), "recent"),
         (dict(first=-1), "first"), (dict(recent=5, first=4), "keep=8"), (dict(recent=1 << 31 - 1, first=1 << 30), "keep=8"),
         (dict(keep=193), "193"), (dict(out_weights=A), "out_weights")]


@pytest.mark.parametrize("kw,text", EVICT)
def test_bad_eviction_is_refused(kw, text):
    d = dict(weights=A, ldw=192, cap=192, keep=8, recent=1, first=1, out_weights=A + 4096, kept=A, layers=2, layer_elems=1 << 20) | kw
    _refused("ssd_paged_evict", (_kv(), d["layers"], d["layer_elems"], _batch(), _batch(), *list(d.values())[:8], None), BAD, text)


@pytest.mark.parametrize("off,ldw", [(4, 192), (-4, 192), (4 * 192, 192), (4 * (3 * 2 * 2 - 1) * 400 + 4 * 191, 400)])
def test_eviction_into_weights_that_overlap_in_part_is_refused(off, ldw):
    """Rows of two layers, three sequences and two kv heads."""
    kv, batch = _kv(kv_heads=2), _batch(n_seq=3)
    _refused("ssd_paged_evict", (kv, 2, 1 << 20, batch, batch, A, ldw, 192, 8, 1, 1, A + off, A, None), BAD, "overlap")


def test_eviction_into_too_few_pages_or_another_batch_is_refused():
    call = lambda after, keep: (_kv(), 1, 1 << 20, _batch(), after, A, 192, 192, keep, 1, 1, A + 4096, A, None)  # noqa: E731
    _refused("ssd_paged_evict", call(_batch(table_cols=1), 65), BAD, "new table")
    _refused("ssd_paged_evict", call(_batch(n_seq=3), 8), BAD, "sequences")


LOGPROBS = [(dict(logits=None), BAD, "null"), (dict(tokens=None), BAD, "null"), (dict(rank=None), BAD, "null"), (dict(top_ids=None), BAD, "null"),
            (dict(M=-1), BAD, "M=-1"), (dict(V=0), BAD, "V=0"), (dict(V=1 << 25, ld=1 << 25), RANGE, "2^24"), (dict(dtype=3), BAD, "dtype"),
            (dict(top=-1), BAD, "alternatives"), (dict(top=33), RANGE, "alternatives"), (dict(top=20, V=10), BAD, "alternatives"),
            (dict(ld=50000), BAD, "stride"), (dict(logits=A + 1), BAD, "aligned"), (dict(ws=None), BAD, "workspace"),
            (dict(ws=A + 8), BAD, "workspace"), (dict(ws_bytes=10), BAD, "workspace")]


@pytest.mark.parametrize("kw,code,text", LOGPROBS)
def test_bad_logprobs_are_refused(kw, code, text):
    d = dict(logits=A, dtype=0, ld=128256, M=3, V=128256, tokens=A, tokens64=0, top=5, ws=A, ws_bytes=1 << 20, logprobs=A, entropy=A, rank=A,
             top_ids=A, top_logprobs=A) | kw
    _refused("ssd_token_logprobs", (*d.values(), None), code, text)


def test_a_prompt_call_that_cuts_the_length_needs_its_workspace():
    from ssd import ops

    b = _batch(table_cols=128, ld_table=128)
    assert ops.paged_prompt_ws_floats(4, 4, 2, 64, 2, 8192) > 0 and ops.paged_prompt_ws_floats(4, 4, 2, 64, 2, 400) == 0
    assert ops.paged_prompt_ws_floats(8192, 32, 8, 128, 1, 8192) == 0
    call = lambda ws, n: (_kv(), b, A, 256, 4, 4, 8192, 0.1, ws, n, A, 256, None)  # noqa: E731
    for ws, n in ((None, 1 << 20), (A, 100), (A + 4, 1 << 20)):
        _refused("ssd_paged_prompt_bf16", call(ws, n), BAD, "workspace")


def test_workspace_sizes():
    from ssd import ops

    assert ops.paged_attn_ws_floats(3, 32, 128, 4096, 128) == 3 * 32 * 8 * 130
    assert ops.paged_attn_ws_floats(1, 1, 64, 100, 64, True) == 66 + 2 + 128  # scores start on 16 bytes
    assert ops.token_logprobs_ws_bytes(2000, 128256, torch.bfloat16, 5) == 0  # a workgroup a row
    assert ops.token_logprobs_ws_bytes(1, 128256, torch.bfloat16, 5) > 0
    with pytest.raises(ValueError):
        ops.paged_attn_ws_floats(1, 32, 128, 4096, 100)
    with pytest.raises(ValueError):
        ops.token_logprobs_ws_bytes(1, 0, torch.bfloat16)
    with pytest.raises(ValueError, match="float64"):
        ops.token_logprobs_ws_bytes(1, 100, torch.float64)


def test_python_refusals_without_a_gpu():
    from ssd.engine.kv_cache import PagedBatch, PagedKVCache

    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="table"):
        PagedBatch(torch.zeros(2, 3, **i32), torch.zeros(2, **i32))
    for kw in (dict(head_dim=32), dict(pages=0), dict(kv_heads=0), dict(num_slots=0), dict(span=96), dict(span=8192)):
        with pytest.raises(ValueError):
            PagedKVCache(**(dict(num_slots=1, pages=4, kv_heads=2, head_dim=64, device="cpu") | kw))


def test_page_counts():
    from ssd.engine.kv_cache import PagedKVCache

    cache = PagedKVCache(1, 5, 2, 64, "cpu")
    assert [PagedKVCache.pages_for(n) for n in (0, 1, 64, 65)] == [0, 1, 1, 2]
    a = cache.alloc(2)
    b = cache.alloc(3)
    assert sorted(a + b) == list(range(5)) and cache.free_pages == 0 and cache.alloc(0) == []
    with pytest.raises(RuntimeError, match="overflow"):
        cache.alloc(1)
    cache.free(a)
    for bad in (a[:1], [9], [-1], [b[0], b[0]]):
        with pytest.raises(ValueError, match="in use"):
            cache.free(bad)
    assert cache.free_pages == 2 and sorted(cache.alloc(2)) == sorted(a)
    with pytest.raises(ValueError):
        cache.alloc(-1)
