"""The 8-bit paged cache without a GPU: the reference's quantiser against torch's, and what both entry points refuse."""
import ctypes

import numpy as np
import pytest
import torch

import kv8_reference as ref
from glm_asr_stack_b200 import _lib, engine, ops


def test_reference_codes_are_e4m3():
    got = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.nan_to_num(got, nan=-1e9), np.nan_to_num(ref.VALUE, nan=-1e9))
    x = np.concatenate([np.random.default_rng(0).normal(size=4000) * 2.0 ** np.random.default_rng(1).integers(-12, 9, 4000), ref.VALUE[:127],
                        (ref.VALUE[:126] + ref.VALUE[1:127]) / 2])
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.e4m3(x.astype(np.float32).astype(np.float64)), want)


@pytest.mark.parametrize("amax,want", [(448.0, 1.0), (448.0 * (1 + 2 ** -20), 2.0), (449.0, 2.0), (224.0, 0.5), (0.0, 2.0 ** -126), (1e-40, 2.0 ** -126)])
def test_reference_scale(amax, want):
    assert ref.scale_of(amax) == want
    assert amax <= 448 * want and (want == 2.0 ** -126 or amax > 224 * want)


def _c_cache(**change):
    """Pointers that nothing follows: every case below is refused, or has nothing to do, before a launch."""
    f = {"k": 4096, "v": 8192, "k_scale": 4096, "v_scale": 4096, "num_blocks": 4, "block_size": 16, "kv_heads": 2, "head_dim": 128}
    f.update(change)
    return _lib.Kv8Cache(*[f[n] for n, _ in _lib.Kv8Cache._fields_])


BAD_CACHES = [{"k": 0}, {"v": 0}, {"k_scale": 0}, {"v_scale": 0}, {"k": 4100}, {"v": 4104}, {"k_scale": 4098}, {"num_blocks": 0}, {"block_size": 0},
              {"block_size": 24}, {"kv_heads": 0}, {"head_dim": 64}, {"num_blocks": 1 << 28, "block_size": 16}]


def _append(cache, key=4096, ldk=256, value=4096, ldv=256, query=None, ldq=0, out=None, ldo=0, heads=0, tables=4096, max_blocks=4, lens=4096,
            cu=4096, seqs=1, rows=2, theta=1e4):
    return _lib.load().glmasr_kv8_append(ctypes.byref(cache) if cache is not None else None, key, ldk, value, ldv, query, ldq, out, ldo, heads, tables,
                                         max_blocks, lens, cu, seqs, rows, theta)


def _attend(cache, out=4096, ldo=1024, query=8192, ldq=1024, tables=4096, max_blocks=4, lens=4096, cu=4096, seqs=1, rows=2, heads=8, max_new=2, max_len=9,
            window=0, sinks=0, scale=0.1, ws=4096, ws_bytes=0):
    return _lib.load().glmasr_kv8_attention(out, ldo, query, ldq, ctypes.byref(cache) if cache is not None else None, tables, max_blocks, lens, cu, seqs, rows,
                                            heads, max_new, max_len, window, sinks, scale, ws, ws_bytes)


@pytest.mark.parametrize("change", BAD_CACHES)
def test_both_refuse_the_cache(change):
    assert _append(_c_cache(**change)) == -1
    assert _attend(_c_cache(**change)) == -1


@pytest.mark.parametrize("change", [{"key": 0}, {"key": 4098}, {"ldk": 252}, {"ldk": 128}, {"value": 0}, {"ldv": 255}, {"theta": -1.0}, {"theta": float("nan")},
                                    {"theta": float("inf")}, {"seqs": -1}, {"rows": -1}, {"max_blocks": 0}, {"tables": 0}, {"lens": 0}, {"cu": 4097},
                                    {"query": 4096, "ldq": 1024, "heads": 8}, {"out": 4096, "ldo": 1024}, {"query": 4096, "ldq": 1024, "out": 4096, "ldo": 1024, "heads": 0},
                                    {"query": 4096, "ldq": 1020, "out": 4096, "ldo": 1024, "heads": 8}, {"query": 4096, "ldq": 512, "out": 4096, "ldo": 1024, "heads": 8}])
def test_append_refuses(change):
    assert _append(_c_cache(), **change) == -1
    assert _append(None) == -1


@pytest.mark.parametrize("change", [{"out": 0}, {"query": 0}, {"out": 4104}, {"ldo": 1020}, {"ldq": 512}, {"heads": 0}, {"heads": 7}, {"max_new": -1}, {"max_len": -1},
                                    {"window": -1}, {"sinks": -1}, {"scale": float("nan")}, {"scale": -1.0}, {"scale": float("inf")}, {"seqs": -1}, {"rows": -1},
                                    {"max_blocks": 0}, {"tables": 0}, {"lens": 4097}, {"ws": 0}])
def test_attention_refuses(change):
    assert _attend(_c_cache(), **change) == -1
    assert _attend(None) == -1


def test_nothing_to_do_is_no_error():
    assert _append(_c_cache(), seqs=0, rows=0) == 0 and _append(_c_cache(), rows=0) == 0
    assert _attend(_c_cache(), seqs=0, rows=0) == 0 and _attend(_c_cache(), rows=0) == 0


def test_python_refuses_host_tensors_and_bad_pools():
    pool = engine.KV8Pool(2, 16, 1, 2, device="cpu")
    z = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv8_append(*pool.layer(0), z, z, i[:1].view(1, 1), i[:1], i)
    with pytest.raises(ValueError):
        ops.kv8_attention(z, *pool.layer(0), i[:1].view(1, 1), i[:1], i)
    for size in (0, -16, 8, 24):
        with pytest.raises(ValueError):
            engine.KV8Pool(2, size, 1, 2, device="cpu")
