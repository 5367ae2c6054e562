"""The C entry points of the 8-bit paged cache without a GPU: kv8_api.cu is host code, compiled here against launches that only
count, so that a call with good arguments returns 0 and every refusal shows the check it is for."""
import ctypes
import os
import random
import subprocess
import sys

import pytest

from conftest import ROOT
from glm_asr_stack_b200 import _lib

CSRC = os.path.join(ROOT, "glm_asr_stack_b200", "csrc")
FAKES = r"""
#include "kv8_attention.cuh"
#include "runtime.cuh"
namespace glmasr {
static int launched = 0;
static Kv8Attend last;
cudaStream_t current_stream() { return nullptr; }
void note_launches(int) {}
size_t kv8_attention_workspace_bytes() { return 4096; }
bool kv8_append_launch(uint8_t *, uint8_t *, float *, float *, const __nv_bfloat16 *, long long, const __nv_bfloat16 *, long long, const __nv_bfloat16 *,
                       long long, __nv_bfloat16 *, long long, const Kv8Batch &, double, cudaStream_t) { ++launched; return true; }
bool kv8_attention_launch(const Kv8Attend &a, int, int, void *, cudaStream_t, int &n) { ++launched; last = a; n = 1; return true; }
}
extern "C" cudaError_t cudaGetLastError() { return cudaSuccess; }
int kv8_looks = 0, device = 0;
namespace glmasr { int kv8_take_status() { ++kv8_looks; return 5; } }
extern "C" cudaError_t cudaGetDevice(int *d) { *d = device; return device < 0 ? cudaErrorNoDevice : cudaSuccess; }
extern "C" int status(int on) { device = on; return glmasr::kv8_status(); }
extern "C" int looks() { return kv8_looks; }
extern "C" int launches() { return glmasr::launched; }
"""
A = 1 << 20            # addresses that nothing follows


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("kv8_entry")
    (tmp / "fakes.cpp").write_text(FAKES)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", CSRC, "-I", os.path.join(cuda, "include"), "-o", str(tmp / "e.so"),
                    str(tmp / "fakes.cpp"), "-x", "c++", os.path.join(CSRC, "kv8_api.cu")], check=True, capture_output=True)
    dll = ctypes.CDLL(str(tmp / "e.so"))
    for name in ("glmasr_kv8_append", "glmasr_kv8_attention", "glmasr_kv8_attention_workspace"):
        getattr(dll, name).restype, getattr(dll, name).argtypes = _lib.SIGNATURES[name]
    return dll


CACHE = {"k": A, "v": A, "k_scale": A, "v_scale": A, "num_blocks": 4, "block_size": 16, "kv_heads": 2, "head_dim": 128}
APPEND = dict(key=A, ldk=256, value=A, ldv=256, query=2 * A, ldq=1024, out=3 * A, ldo=1024, heads=8, tables=A, max_blocks=4, lens=A, cu=A, seqs=1,
              rows=2, theta=1e4)
ATTEND = dict(out=A, ldo=1024, query=2 * A, ldq=1024, tables=A, max_blocks=4, lens=A, cu=A, seqs=1, rows=2, heads=8, max_new=2, max_len=9, window=0,
              sinks=0, scale=0.1, ws=A, ws_bytes=4096)


def append(lib, cache=CACHE, launches=1, **change):
    f = {**APPEND, **change}
    c = ctypes.byref(_lib.Kv8Cache(*[cache[n] for n, _ in _lib.Kv8Cache._fields_])) if cache is not None else None
    before = lib.launches()
    code = lib.glmasr_kv8_append(c, *f.values())
    assert lib.launches() - before == (launches if code == 0 else 0)
    return code


def attend(lib, cache=CACHE, launches=1, **change):
    f = {**ATTEND, **change}
    c = ctypes.byref(_lib.Kv8Cache(*[cache[n] for n, _ in _lib.Kv8Cache._fields_])) if cache is not None else None
    before = lib.launches()
    code = lib.glmasr_kv8_attention(f["out"], f["ldo"], f["query"], f["ldq"], c, *list(f.values())[4:])
    assert lib.launches() - before == (launches if code == 0 else 0)
    return code


def elements(address, ld, heads, rows):
    return {address // 2 + r * ld + i for r in range(rows) for i in range(0, heads * 128, 8)}


def test_outputs_that_overlap_inputs_are_refused(lib):
    """Against the sets of elements, for rows at one pitch; shifted by rows, by heads and by 16 bytes."""
    rng = random.Random(0)
    refused = 0
    for _ in range(4000):
        heads, rows, ld = 8, rng.randint(1, 5), rng.choice([1024, 1032, 1536, 2048, 4096])
        shift = 2 * rng.choice([rng.randint(-6, 6) * ld, rng.randint(-6, 6) * ld + rng.choice([-1, 1]) * rng.choice([8, 128, 512, 1016, 1024, ld - 1024]),
                                8 * rng.randint(-4000, 4000)])
        want = bool(elements(A, ld, heads, rows) & elements(A + shift, ld, heads, rows))
        assert attend(lib, out=A, ldo=ld, query=A + shift, ldq=ld, rows=rows) == (-1 if want else 0), (rows, ld, shift)
        far = {"key": 64 * A, "value": 64 * A}
        assert append(lib, query=A + shift, ldq=ld, out=A, ldo=ld, rows=rows, **far) == (-1 if want and shift != 0 else 0), (rows, ld, shift)
        for which, pitch in (("key", "ldk"), ("value", "ldv")):
            hit = bool(elements(A, ld, heads, rows) & elements(A + shift, ld, 2, rows))
            assert append(lib, **{**far, "query": 32 * A, "ldq": ld, "out": A, "ldo": ld, "rows": rows, which: A + shift, pitch: ld}) == (-1 if hit else 0)
        refused += want
    assert 500 < refused < 3500


def test_outputs_at_another_pitch_have_to_lie_apart(lib):
    assert attend(lib, out=A, ldo=1024, query=A, ldq=2048) == -1
    assert attend(lib, out=A, ldo=2048, query=A + 2048, ldq=1024) == -1         # between the rows, but for one array's sake
    assert attend(lib, out=A, ldo=1024, query=A + 4 * 1024, ldq=2048) == 0
    assert attend(lib, out=A + 2 * (2048 + 1024), ldo=1024, query=A, ldq=2048) == 0
    assert attend(lib, out=A, ldo=8, query=A + 2048, ldq=16, rows=1) == 0       # one row has no pitch
    assert append(lib, query=A, ldq=1024, out=A, ldo=2048) == -1
    assert append(lib, query=A, ldq=1024, out=A, ldo=2048, rows=1, key=64 * A, value=64 * A) == 0
    assert append(lib, query=A, ldq=1536, out=A, ldo=1536, key=A + 2048, ldk=1536, value=A + 2560, ldv=1536) == 0       # one fused projection


def test_tensor_memory_is_asked_for_between_the_wait_and_the_signal():
    """An allocation of tensor memory waits without a limit: only when all earlier kernels are done, and later ones may not start before
    every warp of the block knows that it has come."""
    kernels = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.startswith("kv8_") or not name.endswith(".cu"):
            continue
        for body in open(os.path.join(CSRC, name)).read().split("__global__")[1:]:
            if "tmem_alloc(" not in body:
                continue
            kernels += 1
            alloc = body.index("tmem_alloc(")
            assert body.count("tmem_alloc(") == 1 and body.count("pdl_launch_dependents();") == 1 and "pdl_wait();" in body[:alloc], name
            signal = body.index("pdl_launch_dependents();")
            assert "__syncthreads();" in body[alloc:signal], name
    assert kernels == 2


def test_the_status_of_a_device_without_such_a_launch_is_not_asked_for(lib):
    assert attend(lib) == 0 and lib.status(0) == 5            # this device has one
    before = lib.looks()
    assert lib.status(1) == 0 and lib.status(2) == 0 and lib.looks() == before
    assert append(lib) == 0 and lib.status(2) == 0            # an append waits for nothing
    assert attend(lib, ws=0) == -1 and lib.status(2) == 0 and lib.looks() == before
    assert attend(lib) == 0 and lib.status(2) == 5 and lib.status(1) == 0 and lib.looks() == before + 1
    lib.status(0)


BAD_CACHES = [{"k": 0}, {"v": 0}, {"k_scale": 0}, {"v_scale": 0}, {"k": A + 4}, {"v": A + 8}, {"k_scale": A + 2}, {"v_scale": A + 1}, {"num_blocks": 0}, {"num_blocks": -1},
              {"block_size": 0}, {"block_size": -16}, {"block_size": 24}, {"kv_heads": 0}, {"kv_heads": -2}, {"head_dim": 64}, {"head_dim": 256},
              {"num_blocks": 1 << 26}, {"num_blocks": 1 << 16, "block_size": 1 << 14}]
BAD_BATCHES = [{"tables": 0}, {"tables": A + 2}, {"lens": 0}, {"lens": A + 1}, {"cu": 0}, {"cu": A + 3}, {"seqs": -1}, {"rows": -1}, {"max_blocks": 0}, {"max_blocks": -1}]


def test_good_calls_are_launched(lib):
    assert append(lib) == 0 and attend(lib) == 0
    assert append(lib, query=None, out=None, heads=0, ldq=0, ldo=0) == 0
    assert append(lib, theta=0.0) == 0 and append(lib, ldk=256 + 8, ldv=512, ldq=1032) == 0
    assert attend(lib, window=1 << 30, sinks=1 << 30, max_new=0, max_len=0, scale=0.0) == 0
    largest = {**CACHE, "num_blocks": (1 << 26) - 1}         # 2^31 - 32 rows of codes
    assert append(lib, largest) == 0 and attend(lib, largest) == 0
    nothing = dict(launches=0, query=None, out=None)          # to do: no error, whatever the rows are
    assert append(lib, rows=0, key=0, value=0, **nothing) == 0 and append(lib, seqs=0, key=0, value=0, **nothing) == 0
    assert attend(lib, rows=0, ws=0, **nothing) == 0 and attend(lib, seqs=0, ws=0, **nothing) == 0


@pytest.mark.parametrize("change", BAD_CACHES)
def test_a_bad_cache_is_refused(lib, change):
    assert append(lib, {**CACHE, **change}) == -1 and attend(lib, {**CACHE, **change}) == -1
    assert append(lib, None) == -1 and attend(lib, None) == -1


@pytest.mark.parametrize("change", BAD_BATCHES)
def test_a_bad_batch_is_refused(lib, change):
    assert append(lib, **change) == -1 and attend(lib, **change) == -1


@pytest.mark.parametrize("change", [{"key": 0}, {"key": A + 2}, {"ldk": 252}, {"ldk": 128}, {"ldk": -256}, {"value": 0}, {"value": A + 8}, {"ldv": 255}, {"ldv": 248},
                                    {"theta": -1.0}, {"theta": float("nan")}, {"theta": float("inf")}, {"query": None}, {"out": None}, {"heads": 0}, {"heads": -8},
                                    {"query": 2 * A + 8}, {"ldq": 1020}, {"ldq": 512}, {"out": 3 * A + 4}, {"ldo": 1028}, {"ldo": 1016}])
def test_append_refuses(lib, change):
    assert append(lib, **change) == -1


@pytest.mark.parametrize("change", [{"out": 0}, {"out": A + 8}, {"ldo": 1020}, {"ldo": 1016}, {"query": 0}, {"query": 2 * A + 2}, {"ldq": 1028}, {"ldq": 512}, {"heads": 0},
                                    {"heads": 7}, {"heads": -2}, {"max_new": -1}, {"max_len": -1}, {"window": -1}, {"sinks": -1}, {"scale": float("nan")},
                                    {"scale": -1.0}, {"scale": float("inf")}, {"ws": 0}, {"ws": A + 8}, {"ws_bytes": 4095}, {"ws_bytes": 0}, {"ws_bytes": -1},
                                    {"rows": 1 << 28, "ldq": 1024, "query": 1 << 50}])
def test_attention_refuses(lib, change):
    assert attend(lib, **change) == -1


def test_a_block_that_gives_up_leaves_nothing_to_join():
    """The second launch reads each block's word on what to join, whatever became of the block: written on every way out."""
    body = open(os.path.join(CSRC, "kv8_attention.cu")).read().split("__global__")[1]
    ways_out = [body[:i] for i in range(len(body)) if body.startswith("        return;\n", i) and "mbar_init" not in body[:i]]
    assert len(ways_out) == 1
    for way in ways_out:
        assert "p.part.join[blockIdx.x].last = -1" in way and way.index("pdl_wait();") < way.index("p.part.join")
    assert "if (leader && !p.whole) p.part.join[blockIdx.x] = join;" in body


def test_without_a_device_the_calls_return(lib):
    """-1, and a workspace of 0 bytes; what asks for the device's size ends the process where there is none."""
    lib.status(-1)
    assert lib.glmasr_kv8_attention_workspace() == 0 and attend(lib) == -1 and lib.status(-1) == 0
    lib.status(0)
    assert lib.glmasr_kv8_attention_workspace() == 4096 and attend(lib) == 0
    code = """if True:
        import ctypes, sys
        sys.path[:0] = [%r, %r]
        from glm_asr_stack_b200 import _lib
        import test_kv8_host as t
        size = _lib.load().glmasr_kv8_attention_workspace()
        print(size, t._append(t._c_cache()), t._attend(t._c_cache(), ws_bytes=1 << 40))
    """ % (ROOT, os.path.join(ROOT, "tests"))
    env = {**os.environ, "CUDA_VISIBLE_DEVICES": ""}
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env)
    assert r.returncode == 0 and r.stdout.split() == ["0", "-1", "-1"], (r.stdout, r.stderr)
