"""Refusals of the batch-serving operators and their host-side layout; no device call is made."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parent.parent
I32, BF = torch.int32, torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from diffusorrt_b200 import _lib, build

    build.build()
    return _lib.load()


def test_args_struct_matches_header(tmp_path):
    from diffusorrt_b200 import _lib, kernels

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    py = _lib.CacheAttendArgs
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "diffusorrt_b200.h"', "int main(void) {",
             'printf("size %zu\\n", sizeof(drt_cache_attend_args));']
    lines += [f'printf("{f} %zu\\n", offsetof(drt_cache_attend_args, {f}));' for f, _ in py._fields_]
    (tmp_path / "a.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-I", str(ROOT / "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    assert kernels._ATTEND.size == ctypes.sizeof(py)
    for line in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.split("\n")[:-1]:
        name, value = line.split()
        assert int(value) == (ctypes.sizeof(py) if name == "size" else getattr(py, name).offset), name


def test_constants_match_header():
    from diffusorrt_b200 import _lib

    defines = dict(re.findall(r"#define (DRT_\w+) (\d+)", (ROOT / "include" / "diffusorrt_b200.h").read_text()))
    for name in ("CODE_INT8", "CODE_E4M3", "TYPE_F32", "TYPE_BF16", "TYPE_F16"):
        assert int(defines["DRT_" + name]) == getattr(_lib, name)


def refuse(lib, status, text, message):
    assert status in (2, 3), status
    assert message in lib.drt_last_error().decode(), lib.drt_last_error()


P = 4096  # an aligned address that nothing may touch


def plan(lib, **change):
    a = dict(start=P, count=P, held=P, held_out=P, requests=2, tables=P, ld=4, width=4, block=16, ring=P, size=8, rin=P, rout=P,
             rs=P, slots=P, pos=P, rows=5, lengths=P, status=P)
    a.update(change)
    return lib.drt_cache_plan(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(start=None), "null"), (dict(status=None), "null"), (dict(ring=None), "null"), (dict(slots=None), "slots"),
    (dict(requests=-1), "requests"), (dict(rows=-1), "max_rows"), (dict(ld=3), "table"), (dict(width=0), "table"),
    (dict(block=0), "table"), (dict(width=1 << 27, ld=1 << 27, block=128), "2^31"), (dict(size=0), "capacity")])
def test_plan_refusals(lib, change, message):
    refuse(lib, plan(lib, **change), "plan", message)


def append(lib, **change):
    a = dict(k=P, kr=256, kh=128, v=P, vr=256, vh=128, dtype=1, rows=3, slots=P, kc=P, vc=P, ks=P, vs=P, blocks=4, heads=2, block=16,
             dim=128, code=0)
    a.update(change)
    return lib.drt_cache_append(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(k=None), "null"), (dict(kc=None), "null"), (dict(vs=None), "null"), (dict(rows=-1), "rows"), (dict(dtype=0), "bf16"),
    (dict(dtype=7), "bf16"), (dict(block=17), "block"), (dict(block=256), "block"), (dict(dim=96), "dim"), (dict(code=2), "code"),
    (dict(heads=0), "geometry"), (dict(blocks=0), "geometry"), (dict(blocks=1 << 28), "2^31"), (dict(kc=P + 8), "aligned")])
def test_append_refusals(lib, change, message):
    refuse(lib, append(lib, **change), "append", message)


def read(lib, **change):
    a = dict(slots=P, rows=3, kc=P, vc=P, ks=P, vs=P, blocks=4, heads=2, block=16, dim=128, code=0, ko=P, vo=P, dtype=1)
    a.update(change)
    return lib.drt_cache_read(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(slots=None), "null"), (dict(ko=None), "null"), (dict(dtype=3), "bf16"), (dict(rows=-2), "rows"), (dict(vo=P + 4), "aligned"),
    (dict(block=48), "block")])
def test_read_refusals(lib, change, message):
    refuse(lib, read(lib, **change), "read", message)


def attend(lib, **change):
    from diffusorrt_b200 import _lib

    a = dict(q=P, q_row=512, q_head=128, out=P, out_row=512, out_head=128, k_cache=P, v_cache=P, k_scale=P, v_scale=P, blocks=4,
             tables=P, ld_tables=4, lengths=P, row_start=P, scratch=P, q_rows=3, heads=4, kv_heads=2, dim=128, dtype=1, code=0,
             block=16, width=4, requests=2, mask_block=1, scale=0.1)
    a.update(change)
    return lib.drt_cache_attend(ctypes.byref(_lib.CacheAttendArgs(**a)), None)


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "null"), (dict(scratch=None), "null"), (dict(tables=None), "null"), (dict(dtype=0), "bf16"),
    (dict(heads=5), "multiple"), (dict(heads=0), "multiple"), (dict(kv_heads=0), "geometry"), (dict(requests=-1), "requests"),
    (dict(requests=20000), "requests"), (dict(width=0), "table"), (dict(ld_tables=3), "table"), (dict(mask_block=-1), "mask_block"),
    (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"), (dict(out=P + 2), "out"), (dict(out_head=127), "out"),
    (dict(scratch=P + 4), "scratch"), (dict(q_rows=-1), "requests"), (dict(q_rows=1 << 30), "2^31")])
def test_attend_refusals(lib, change, message):
    refuse(lib, attend(lib, **change), "attend", message)


def score(lib, **change):
    a = dict(logits=P, dtype=0, ld=100, logit_rows=2, index=None, rows=2, vocab=100, tokens=P, temperature=0.0, exclude=-1, top=2, scratch=P, lp=P,
             ent=P, rank=P, tt=P, tl=P)
    a.update(change)
    return lib.drt_selector_logprobs(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(logits=None), "null"), (dict(scratch=None), "null"), (dict(tt=None), "null"), (dict(tokens=None), "tokens"),
    (dict(dtype=5), "logits"), (dict(top=33), "top"), (dict(top=-1), "top"), (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=1e-31), "temperature"),
    (dict(exclude=100), "exclude"), (dict(ld=99), "geometry"), (dict(vocab=0), "geometry"), (dict(rows=-1), "geometry"),
    (dict(logits=P + 2), "misaligned"), (dict(logit_rows=1), "more rows"), (dict(logit_rows=0, index=P), "more rows")])
def test_score_refusals(lib, change, message):
    refuse(lib, score(lib, **change), "score", message)


def test_calls_without_work_touch_nothing(lib):
    assert append(lib, rows=0, k=None, v=None, slots=None) == 0
    assert read(lib, rows=0, slots=None) == 0
    assert attend(lib, q_rows=0, q=None) == 0
    assert attend(lib, requests=0, lengths=None) == 0
    assert score(lib, rows=0, logits=None) == 0


def test_python_checks_come_before_the_library():
    """Tensors on the CPU, of other types, shapes or layouts are refused by name."""
    from diffusorrt_b200 import kernels

    k = torch.zeros(2, 1, 64, dtype=BF)
    cache = (torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 1, 64, 16, dtype=torch.int8), torch.zeros(2, 1),
             torch.zeros(2, 1))
    slots = torch.zeros(2, dtype=I32)
    for call in (lambda: kernels.append_cache_q8(k, k, slots, *cache), lambda: kernels.read_cache_q8(slots, *cache),
                 lambda: kernels.plan_cache(slots, slots, slots, torch.zeros(2, 3, dtype=I32), slots, slots, block_size=16, max_rows=1),
                 lambda: kernels.attend_cache_q8(k, *cache, torch.zeros(1, 3, dtype=I32), slots[:1], slots),
                 lambda: kernels.select_logprobs(torch.zeros(2, 9), slots)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    dev = -1  # the CPU
    with pytest.raises(ValueError, match="int8 or float8"):
        kernels._cache_args(cache[0].to(torch.uint8), *cache[1:], dev)
    with pytest.raises(ValueError, match="16, 32, 64 or 128"):
        kernels._cache_args(torch.zeros(2, 1, 24, 64, dtype=torch.int8), *cache[1:], dev)
    with pytest.raises(ValueError, match="v_cache"):
        kernels._cache_args(cache[0], torch.zeros(2, 1, 16, 64, dtype=torch.int8), *cache[2:], dev)
    with pytest.raises(ValueError, match="k_scale"):
        kernels._cache_args(cache[0], cache[1], torch.zeros(2, 2), cache[3], dev)
    with pytest.raises(ValueError, match="contiguous"):
        kernels._cache_args(cache[0].transpose(2, 3), *cache[1:], dev)
    with pytest.raises(ValueError, match="int8 or float8"):
        kernels.cache_q8(2, 1, 16, dtype=BF, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        kernels._check_ints(torch.zeros(4, dtype=torch.int64), "slots", dev)
    assert kernels._cache_args(*kernels.cache_q8(2, 3, 32, 64, dtype=torch.float8_e4m3fn, device="cpu"), dev) == (2, 3, 32, 64, 1)


def test_plan_oracle_on_hand_cases():
    import sys

    sys.path.insert(0, str(ROOT / "tests"))
    import cache_q8_oracle as oracle

    p = oracle.plan([10, 0, 7], [8, -1, 0], [1, 2, 1], [[5, -1], [6, 7], [8, -1]], [0, 1, 2, 3, 4, 9, 9, 9, 9], [3, 2], 16, 9)
    assert p["tables"][0] == [5, 3] and p["held"] == [2, 0, 1] and p["ring_state"] == [4, 3]
    assert p["ring"][5:7] == [6, 7] and p["row_start"] == [0, 8, 8, 8] and p["lengths"] == [18, 0, 7]
    assert p["slots"] == [5 * 16 + i for i in range(10, 16)] + [48, 49, -1] and p["status"] == 0
    assert oracle.limit(5, 20, 4, 0) == 8 and oracle.limit(5, 7, 4, 0) == 7 and oracle.limit(2, 20, 4, 6) == 6
    assert oracle.limit(6, 20, 4, 6) == 10 and oracle.limit(-1, 20, 0, 0) == 0 and oracle.limit(3, 20, 0, 9) == 20
