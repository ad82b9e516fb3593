"""The 8-bit cache without a GPU: what the entry points refuse, sizes, allocation, and the reference that the GPU tests compare with."""

import numpy as np
import pytest
import torch

import quantized_reference as R
from nano_vllm_jax_b200 import _lib
from nano_vllm_jax_b200 import kv_cache as kvc
from nano_vllm_jax_b200.backends import B200Backend, full_attention_kv_cache_dtype
from nano_vllm_jax_b200.kernels import paged_kv, quantized_kv as Q

INVALID, UNSUPPORTED, TOO_LARGE = -1, -2, -5
P = 1 << 20  # stands for a pointer: the calls below are refused before anything is launched


def _append(**change):
    a = dict(new_k=P, new_v=P, dtype=0, positions=P, tables=P, ids=None, table_rows=2, width=4, qsl=None, qsl_rows=0, lens=None, rows=2,
             cols=3, k=P, v=P, ks=P, vs=P, blocks=8, bs=16, hkv=2, d=256, status=P) | change
    return _lib.load().nvj_kv_append_quantized(*a.values(), None)


def _decode(**change):
    a = dict(q=P, dtype=0, k=P, v=P, ks=P, vs=P, blocks=8, bs=16, hkv=2, d=256, hq=8, tables=P, width=4, lens=P, pos=None, qsl=None, rows=2,
             tokens=1, scale=1.0, out=P, status=P, ws=None, nbytes=0, form=0) | change
    return _lib.load().nvj_paged_decode_quantized(*a.values(), None)


def _prefill(**change):
    a = dict(q=P, dtype=0, k=P, v=P, ks=P, vs=P, blocks=8, bs=16, hkv=2, d=256, hq=8, tables=P, width=4, lens=P, pos=P, qsl=P, rows=2,
             bucket=5, scale=1.0, out=P, status=P, ws=None, nbytes=0, singles=0, pairs=-1) | change
    return _lib.load().nvj_paged_prefill_quantized(*a.values(), None)


def _layout(**change):
    a = dict(cached=P, new=P, rows=2, tables=P, width=4, bs=16, free=P, count=9, head=P, bucket=8, pos=P, ids=P, slots=P, qsl=P, lens=P,
             head_out=P + 64, status=P) | change
    return _lib.load().nvj_build_packed_layout(*a.values(), None)


@pytest.mark.parametrize("call", [_append, _decode, _prefill])
@pytest.mark.parametrize("change,code", [
    ({"d": 96}, UNSUPPORTED), ({"d": 512}, UNSUPPORTED), ({"bs": 8}, UNSUPPORTED), ({"bs": 80}, UNSUPPORTED), ({"bs": 24}, UNSUPPORTED),
    ({"hkv": 0}, UNSUPPORTED), ({"dtype": 3}, UNSUPPORTED), ({"dtype": -1}, UNSUPPORTED), ({"k": P + 8}, INVALID), ({"v": None}, INVALID),
    ({"ks": None}, INVALID), ({"status": None}, INVALID), ({"blocks": -1}, INVALID), ({"width": -1}, INVALID), ({"rows": -1}, INVALID)])
def test_calls_that_every_entry_point_refuses(call, change, code):
    assert call(**change) == code


@pytest.mark.parametrize("change,code", [
    ({"new_k": P + 4}, INVALID), ({"positions": None}, INVALID), ({"tables": None}, INVALID), ({"width": 0}, INVALID), ({"blocks": 0}, INVALID),
    ({"ids": P}, INVALID), ({"rows": 1 << 16, "cols": 1 << 16}, TOO_LARGE)])
def test_appends_that_are_refused(change, code):
    assert _append(**change) == code


@pytest.mark.parametrize("change,code", [
    ({"hq": 9}, INVALID), ({"hq": 0}, INVALID), ({"q": P + 2}, INVALID), ({"out": P + 4}, INVALID), ({"lens": None}, INVALID),
    ({"qsl": P, "tokens": 2}, INVALID), ({"qsl": P, "pos": None}, INVALID), ({"width": 1 << 27}, TOO_LARGE),
    ({"tokens": 1 << 15}, TOO_LARGE), ({"form": 3}, INVALID), ({"form": -1}, INVALID)])
def test_decode_calls_that_are_refused(change, code):
    assert _decode(**change) == code


@pytest.mark.parametrize("change,code", [
    ({"hq": 9}, INVALID), ({"pos": None}, INVALID), ({"qsl": None}, INVALID), ({"lens": None}, INVALID), ({"bucket": -1}, INVALID),
    ({"bucket": 1 << 29}, TOO_LARGE)])
def test_prefill_calls_that_are_refused(change, code):
    assert _prefill(**change) == code


@pytest.mark.parametrize("change,code", [
    ({"rows": -1}, INVALID), ({"bs": 0}, INVALID), ({"head": None}, INVALID), ({"head_out": P}, INVALID), ({"cached": None}, INVALID),
    ({"free": None}, INVALID), ({"pos": None}, INVALID), ({"rows": 16385}, TOO_LARGE), ({"width": 1 << 27}, TOO_LARGE)])
def test_layouts_that_are_refused(change, code):
    assert _layout(**change) == code


def test_calls_with_nothing_to_do_launch_nothing():
    assert _append(rows=0) == 0 and _append(cols=0) == 0
    assert _decode(rows=0) == 0 and _decode(tokens=0) == 0
    assert _prefill(bucket=0) == 0


def test_scratch_of_a_prefill():
    size = _lib.load().nvj_paged_prefill_quantized_workspace_bytes
    # (q type, rows, table width, block size, kv heads, head_dim, query heads, scale, single rows, tokens, 64-token tiles)
    page = 16 * 2 * 256 * 2
    assert size(0, 3, 100, 16, 2, 256, 8, 0.1, 0, 64, -1) == 300 * 2 * page + 1280
    sums = 4 * 8 * 2 * 128 * 256 * 4  # long rows of few tokens: what a cluster's CTAs have summed
    assert size(0, 1, 32768, 16, 2, 256, 8, 0.1, 0, 64, -1) > sums and size(0, 1, 32769, 16, 2, 256, 8, 0.1, 0, 64, -1) == sums  # at most 1 GiB
    assert size(1, 1, 1024, 16, 2, 256, 8, 0.1, 0, 64, -1) == sums == size(1, 1, 1024, 16, 2, 256, 8, 0.1, 0, 64, 1)
    assert size(0, 1, 1024, 16, 2, 256, 8, 0.0, 0, 64, -1) == sums
    assert size(1, 1, 512, 16, 2, 256, 8, 0.1, 0, 64, -1) == 0  # not long enough
    assert size(1, 1, 1024, 16, 2, 256, 8, 0.1, 0, 8192, -1) == 0  # tiles enough without clusters
    assert size(1, 1, 1024, 16, 2, 100, 8, 0.1, 0, 64, -1) == 0 and size(1, 0, 1024, 16, 2, 256, 8, 0.1, 0, 64, -1) == 0
    decode = _lib.load().nvj_paged_decode_quantized_workspace_bytes(64, 1, 256, 16, 2, 256, 8, 0)  # (0 without a GPU)
    assert size(1, 64, 256, 16, 2, 256, 8, 0.1, 5, 64, -1) >= decode


def test_wrappers_refuse_tensors_that_are_not_on_a_gpu():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(4, 2)
    i = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        Q.kv_append_quantized(torch.zeros(2, 2, 2, 64), torch.zeros(2, 2, 2, 64), k, k, s, s, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        Q.paged_decode_attention_quantized(torch.zeros(2, 4, 64), k, k, s, s, i, i[0], 1.0)
    with pytest.raises(ValueError, match="CUDA"):
        Q.packed_paged_prefill_attention_quantized(torch.zeros(1, 2, 4, 64), k, k, s, s, i, i[0], i[:1], i[0], 16, 1.0, 2)
    with pytest.raises(ValueError, match="CUDA"):
        paged_kv.build_packed_layout(i[0], i[0], i, i[0], i[0, :1], 16, 8)


def test_allocation_of_an_8_bit_cache(monkeypatch):
    monkeypatch.delenv("NANO_VLLM_JAX_FULL_ATTN_KV_CACHE_DTYPE", raising=False)
    spec = kvc.KVCacheSpec(3, 40, 16, 2, 256, torch.float8_e4m3fn, max_kv_cache_bytes=3 * 10 * (2 * 16 * 2 * 256 + 2 * 2 * 4) + 5)
    assert kvc.estimate_kv_cache_bytes(spec) == 3 * 40 * (2 * 16 * 2 * 256 + 2 * 2 * 4)
    storage = B200Backend(device="cpu").allocate_kv_cache(spec, 1, 1)
    assert isinstance(storage, kvc.QuantizedKVCacheStorage) and storage.k_cache.shape == (3, 10, 16, 2, 256)
    assert storage.k_cache.dtype == torch.float8_e4m3fn and storage.v_scale.shape == (3, 10, 2) and float(storage.k_scale.max()) == 2.0 ** -117
    k, v, ks, vs = storage.layer(2)
    assert k.data_ptr() == storage.k_cache[2].data_ptr() and vs.data_ptr() == storage.v_scale[2].data_ptr()
    assert full_attention_kv_cache_dtype(torch.bfloat16, type("C", (), {"full_attention_kv_cache_dtype": "fp8"})) == torch.float8_e4m3fn
    with pytest.raises(ValueError, match="block_size"):
        kvc.init_quantized_kv_cache(kvc.KVCacheSpec(1, 4, 8, 2, 256), device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        kvc.init_quantized_kv_cache(kvc.KVCacheSpec(1, 4, 16, 2, 96), device="cpu")


def test_the_reference_rounds_as_the_format_does():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(4000) * 2.0 ** rng.integers(-14, 9, 4000), R._MAGNITUDES, -R._MAGNITUDES,
                        (R._MAGNITUDES[1:] + R._MAGNITUDES[:-1]) / 2, [447.9, 448, 463, 464, 1e9, 2.0 ** -10, 2.0 ** -11, 0.0]])
    want = torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.nearest(x), want)
    assert R.nearest(np.array([np.nan, np.inf, -np.inf])).tolist() == [127, 126, 254]


@pytest.mark.parametrize("largest,scale", [(448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (224.1, 1.0), (0.0, 2.0 ** -117), (1e-40, 2.0 ** -117),
                                           (3.38e38, 2.0 ** 119), (1.0, 2.0 ** -8)])
def test_scales_of_the_reference(largest, scale):
    assert R.scale_for(largest) == scale


def test_every_named_barrier_of_the_tcgen05_decode_kernel_has_one_meaning():
    # three groups of 128 threads with a barrier each, one of all groups, one of all warps but the producer's: a barrier that two of them used, with
    # different numbers of threads, would hang after a wait that ran out
    import re
    from pathlib import Path
    text = re.sub(r"//[^\n]*", "", (Path(Q.__file__).parents[1] / "csrc" / "quantized_umma.cuh").read_text())
    ids = {name: int(n) for name, n in re.findall(r"\b(kQuBar\w+) = (\d+)", text)}
    groups = max(int(n) for n in re.findall(r"launch_quantized_umma<T, kDim, \d+, (\d+)>", text))
    used = [ids["kQuBarGroup"] + g for g in range(max(groups, 2))] + [ids["kQuBarAll"], ids["kQuBarQueries"]]
    assert len(set(used)) == len(used) and 0 not in used and max(used) < 16
    meetings = set(re.findall(r"qu_meet_any<([^>]*)>\((\w+),", text)) | set(re.findall(r"(named_bar_sync)\((\w+),", text))
    assert meetings == {("128", "bar"), ("L::kSoftmaxThreads", "kQuBarAll"), ("named_bar_sync", "kQuBarQueries")}
    assert re.search(r"\bbar = kQuBarGroup \+ group;", text)


def test_a_layout_does_not_write_its_lengths_over_those_that_it_reads():
    apart = dict(cached=P, new=P + 4096, tables=P + 8192, lens=P + 12288)
    assert _layout(**apart | {"lens": P}) == INVALID and _layout(**apart | {"lens": P + 4096}) == INVALID


def test_the_pipeline_and_the_step_graph_refuse_an_8_bit_cache_at_once():
    from nano_vllm_jax_b200.engine.resident_decode import DecodeStepGraph, ResidentDecodeMetadata
    from nano_vllm_jax_b200.host_pipeline import HostDecodePipeline
    cache = B200Backend(device="cpu").allocate_kv_cache(kvc.KVCacheSpec(1, 4, 16, 2, 256, torch.float8_e4m3fn), 2, 2)
    with pytest.raises(ValueError, match="8-bit"):
        HostDecodePipeline(B200Backend(device="cpu"), cache, 2, 2, 16, 0.1, 4)
    with pytest.raises(ValueError, match="8-bit"):
        DecodeStepGraph(ResidentDecodeMetadata(2, 2, 16, device="cpu"), cache.k_cache, cache.v_cache, 0, 0.1, 4)


def test_rows_do_not_take_blocks_of_another_size():
    from nano_vllm_jax_b200.engine.device_blocks import DeviceBlockPool
    from nano_vllm_jax_b200.engine.resident_decode import ResidentDecodeMetadata
    with pytest.raises(ValueError, match="block size"):
        ResidentDecodeMetadata(2, 4, 16, device="cpu").reserve(DeviceBlockPool([1, 2], 32, device="cpu"))
