"""The paged key/value cache without a GPU: the arithmetic its kernels and host code share, compiled by itself, and
the refusals of its entry points, which are answered before any GPU work."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest
import torch

from nv_embedding_cache_b200 import capi, kv_cache

ROOT = Path(__file__).resolve().parent.parent
INV = capi.NVE_ERROR_INVALID_ARGUMENT


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    out = tmp_path_factory.mktemp("kv_plan") / "libkv_plan_shim.so"
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
                           f"-I{ROOT / 'nv_embedding_cache_b200' / 'csrc'}", str(ROOT / "tests" / "kv_plan_shim.cpp"),
                           "-o", str(out)])
    lib = C.CDLL(str(out))
    lib.kp_div.argtypes, lib.kp_div.restype = [C.c_uint32, C.c_uint32], C.c_uint32
    lib.kp_range.argtypes, lib.kp_range.restype = [C.c_int32, C.c_int32, C.c_int32, C.c_void_p], None
    return lib


def test_division_by_an_invariant(plan):
    rng = random.Random(1)
    top = (1 << 31) - 1
    divisors = list(range(1, 70)) + [100, 127, 128, 129, 1 << 16, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, top]
    divisors += [rng.randrange(1, 1 << rng.randrange(2, 32)) or 1 for _ in range(200)]
    for d in divisors:
        d = min(d, top)
        for n in {0, 1, d - 1, d, min(d + 1, top), top, top - 1, top // d * d, max(top // d * d - 1, 0),
                  *(rng.randrange(0, top + 1) for _ in range(40))}:
            assert plan.kp_div(n, d) == n // d, (n, d)


@pytest.mark.parametrize("total,n", [(1, 1), (7, 3), (64, 64), (65, 64), (1000, 444), ((1 << 31) - 2, 444), (445, 444), (888, 444)])
def test_runs_cover_every_tile_once_and_name_their_owner(plan, total, n):
    at = 0
    out = (C.c_int32 * 2)()
    for c in range(n):
        plan.kp_range(total, n, c, out)
        assert out[0] == at and out[1] > out[0]                 # in order, without a gap, none empty
        assert total // n <= out[1] - out[0] <= -(-total // n)
        for t in {out[0], (out[0] + out[1] - 1) // 2, out[1] - 1}:
            assert plan.kp_cta(total, n, t) == c
        at = out[1]
    assert at == total


def test_unfinished_units_of_a_run_have_slots_of_their_own(plan):
    """Random batches: a run that has only part of a unit has it first (slot 0) or last (slot 1), and two unfinished
    units never share a slot."""
    rng = random.Random(2)
    out = (C.c_int32 * 2)()
    for _ in range(300):
        units = [rng.choice([1, 1, 2, 3, 8, 40]) for _ in range(rng.randrange(1, 30))]
        total = sum(units)
        n = min(total, rng.randrange(1, 20))
        first = 0
        used = set()
        for tiles in units:
            a, b = plan.kp_cta(total, n, first), plan.kp_cta(total, n, first + tiles - 1)
            for c in range(a, b + 1) if a != b else []:
                plan.kp_range(total, n, c, out)
                assert out[0] < first + tiles and out[1] > first          # has some of it
                slot = (c, plan.kp_slot(out[0], first))
                assert slot not in used
                used.add(slot)
            first += tiles


def test_tiles_of_lengths(plan):
    assert [plan.kp_tiles(x, 64) for x in (0, 1, 63, 64, 65, 128, 129, (1 << 31) - 1)] == [0, 1, 1, 1, 2, 2, 3, 1 << 25]
    assert [plan.kp_tiles(x, 128) for x in (0, 1, 128, 129, (1 << 31) - 1)] == [0, 1, 1, 2, 1 << 24]
    assert [plan.kp_tile_rows(w, b) for w, b in ((8, 2), (64, 2), (72, 2), (128, 2), (256, 2), (128, 1), (136, 1))] == \
        [128, 128, 64, 64, 64, 128, 64]


# ---- refusals ------------------------------------------------------------------------------------
def cache_view(**changes):
    c = capi.KvCache(256, 256, (C.c_int64 * 3)(4096, 256, 4096 * 4), (C.c_int64 * 3)(4096, 256, 4096 * 4), 256, None,
                     None, capi.DTYPE_BFLOAT16, 8, 16, 2, 128, None)
    for k, v in changes.items():
        setattr(c, k, v)
    return c


def rows(**changes):
    r = capi.HeadRows(256, 4096, 512, 256, 512, 256, 2)
    for k, v in changes.items():
        setattr(r, k, v)
    return r


def attend_args(**changes):
    a = capi.KvAttend(capi.DTYPE_BFLOAT16, 1, 4, 256, 1024, 256, 256, 1024, 256, None, 256, 4, 4, 256, 64, 1.0, 0)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def append_args(**changes):
    a = capi.KvAppend(capi.DTYPE_BFLOAT16, 2, rows(), rows(out=None), rows(out=None), None, 256, 4, 4, 1, 256, None,
                      512, 0)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def evict_args(**changes):
    a = capi.KvEvict(1, 256, 4, 4, 256, 64, 512, 2, 2, 32, 4, 8, 256, 512)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def refused(status, word):
    assert status == INV, (status, capi.last_error())
    assert word in capi.last_error(), capi.last_error()


BAD_CACHES = [
    (dict(keys=None), "no keys"), (dict(values=None), "no values"), (dict(dtype=capi.DTYPE_FLOAT32), "FLOAT16"),
    (dict(dtype=capi.DTYPE_QINT8_F32), "FLOAT16"), (dict(num_pages=0), "num_pages"), (dict(num_pages=1 << 31), "num_pages"),
    (dict(page_size=0), "page_size"), (dict(num_heads=0), "num_heads"), (dict(head_width=0), "head_width"),
    (dict(head_width=264), "head_width"), (dict(head_width=36), "16 bytes"), (dict(keys=264), "multiples of 16"),
    (dict(key_strides=(C.c_int64 * 3)(4096, 250, 4096)), "multiples of 16"),
    (dict(value_strides=(C.c_int64 * 3)(-4096, 256, 4096)), "negative"), (dict(key_scale=256), "scales"),
]


@pytest.mark.parametrize("change,word", BAD_CACHES)
def test_caches_that_are_refused(change, word):
    c = cache_view(**change)
    size = C.c_size_t(1 << 30)
    refused(capi.lib.nve_b200_kv_append(C.byref(c), C.byref(append_args()), None), word)
    refused(capi.lib.nve_b200_kv_attend(C.byref(c), C.byref(attend_args()), 256, C.byref(size), None), word)
    refused(capi.lib.nve_b200_kv_evict(C.byref(c), C.byref(evict_args()), None), word)


def test_null_arguments_are_refused():
    c, size = cache_view(), C.c_size_t(0)
    lib = capi.lib
    refused(lib.nve_b200_kv_append(None, C.byref(append_args()), None), "NULL")
    refused(lib.nve_b200_kv_append(C.byref(c), None, None), "NULL")
    refused(lib.nve_b200_kv_attend(C.byref(c), None, None, C.byref(size), None), "NULL")
    refused(lib.nve_b200_kv_attend(C.byref(c), C.byref(attend_args()), None, None, None), "NULL")
    refused(lib.nve_b200_kv_evict(C.byref(c), None, None), "NULL")
    refused(lib.nve_b200_rotary(None, capi.DTYPE_FLOAT32, 64, 1, C.byref(rows()), 1, 0, None), "NULL")


@pytest.mark.parametrize("change,word", [
    (dict(dtype=capi.DTYPE_FLOAT16), "cache's type"), (dict(dtype=capi.DTYPE_FLOAT32), "cache's type"),
    (dict(num_q_heads=3), "multiple"), (dict(num_q_heads=0), "multiple"), (dict(num_sequences=-1), "negative"),
    (dict(max_length=65), "max_length"), (dict(max_length=-1), "max_length"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(page_table=None), "page_table"), (dict(lengths=None), "lengths"),
    (dict(pages_per_sequence=-1), "pages_per_sequence"), (dict(pages_per_sequence=1 << 28), "2^31"),
    (dict(num_sequences=2, page_table_stride=3), "overlap"),
])
def test_attention_that_is_refused(change, word):
    size = C.c_size_t(1 << 30)
    refused(capi.lib.nve_b200_kv_attend(C.byref(cache_view()), C.byref(attend_args(**change)), 256, C.byref(size), None), word)


def test_attention_refuses_weights_that_are_not_kept():
    size = C.c_size_t(1 << 30)
    refused(capi.lib.nve_b200_kv_attend(C.byref(cache_view(weights=None)), C.byref(attend_args(accumulate_weights=1)), 256,
                                        C.byref(size), None), "no weights")


def test_attention_of_no_sequences_is_nothing_to_do():
    size = C.c_size_t(77)
    assert capi.lib.nve_b200_kv_attend(C.byref(cache_view()), C.byref(attend_args(num_sequences=0)), None, C.byref(size), None) == 0
    assert size.value == 0


@pytest.mark.parametrize("change,word", [
    (dict(dtype=capi.DTYPE_FLOAT16), "cache's type"), (dict(num_tokens=-1), "tokens"), (dict(num_tokens=1 << 31), "tokens"),
    (dict(k=rows(num_heads=1)), "heads"), (dict(v=rows(num_heads=3)), "heads"), (dict(k=rows(in_=None)), "NULL"),
    (dict(q=rows(out=None)), "NULL"), (dict(q=rows(in_=257)), "value size"), (dict(v=rows(in_token_stride=3)), "value size"),
    (dict(new_lengths=None), "new_lengths"), (dict(new_lengths=256), "new_lengths"), (dict(num_sequences=3), "multiple"),
    (dict(q=rows(out=256, out_token_stride=1024)), "in place"), (dict(num_sequences=0), "without a sequence"),
])
def test_appends_that_are_refused(change, word):
    refused(capi.lib.nve_b200_kv_append(C.byref(cache_view()), C.byref(append_args(**change)), None), word)


def test_e4m3_rows_are_no_input():
    c = cache_view(dtype=capi.DTYPE_E4M3)
    size = C.c_size_t(1 << 30)
    refused(capi.lib.nve_b200_kv_append(C.byref(c), C.byref(append_args(dtype=capi.DTYPE_E4M3)), None), "FLOAT16")
    refused(capi.lib.nve_b200_kv_attend(C.byref(c), C.byref(attend_args(dtype=capi.DTYPE_E4M3)), 256, C.byref(size), None), "FLOAT16")


@pytest.mark.parametrize("change,word", [
    (dict(budget=0), "budget"), (dict(sinks=-1), "budget"), (dict(sinks=25), "budget"), (dict(recent=1 << 31 - 1), "budget"),
    (dict(new_pages_per_sequence=1), "fewer"), (dict(kept=None), "NULL"), (dict(new_lengths=None), "NULL"),
    (dict(new_page_table=None), "NULL"), (dict(new_lengths=256), "new_lengths"), (dict(max_length=65), "max_length"),
    (dict(num_sequences=2, new_page_table_stride=1), "overlap"), (dict(lengths=None), "lengths"),
])
def test_evictions_that_are_refused(change, word):
    refused(capi.lib.nve_b200_kv_evict(C.byref(cache_view()), C.byref(evict_args(**change)), None), word)


def test_eviction_refuses_a_cache_without_weights():
    refused(capi.lib.nve_b200_kv_evict(C.byref(cache_view(weights=None)), C.byref(evict_args()), None), "no weights")


@pytest.mark.parametrize("change,call,word", [
    (dict(), dict(dtype=capi.DTYPE_E4M3), "FLOAT32"), (dict(), dict(width=0), "width"), (dict(), dict(width=1025), "width"),
    (dict(num_pairs=33), dict(), "num_pairs"), (dict(num_pairs=-1), dict(), "num_pairs"), (dict(num_axes=0), dict(), "num_axes"),
    (dict(positions=None), dict(), "positions"), (dict(inv_freq=None), dict(), "inv_freq"), (dict(), dict(tokens=-1), "tokens"),
    (dict(), dict(groups=0), "groups"), (dict(), dict(groups=3), "groups"),
    (dict(), dict(rows=rows(out=256, out_head_stride=512)), "in place"), (dict(), dict(rows=rows(in_=258)), "value size"),
])
def test_rotations_that_are_refused(change, call, word):
    r = capi.Rotary(256, 8, 1, 1, 256, None, 32, 0, None)
    for k, v in change.items():
        setattr(r, k, v)
    a = dict(dtype=capi.DTYPE_FLOAT32, width=64, tokens=4, rows=rows(), groups=1) | call
    refused(capi.lib.nve_b200_rotary(C.byref(r), a["dtype"], a["width"], a["tokens"], C.byref(a["rows"]), a["groups"], 0, None), word)


def test_python_edge_refuses_host_tensors():
    x = torch.zeros((4, 2, 64))
    with pytest.raises(ValueError, match="on the GPU"):
        kv_cache.RotaryPlan(torch.ones(32))
    with pytest.raises(ValueError, match="on the GPU"):
        kv_cache.rotary(x, None, torch.zeros(4, dtype=torch.int32), None)
    with pytest.raises(ValueError, match="on the GPU"):
        kv_cache.PagedKVCache(torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16), torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16))
