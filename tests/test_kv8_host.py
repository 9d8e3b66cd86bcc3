"""What the 8-bit cache's entry points decide on the host: the sizes of workspaces, refusals of what
a caller can get wrong, and the checks of the Python handles."""
import ctypes as C

import pytest
import torch

import nyion_hip as nh

COUNTERS = 16384


def cache_of(blocks=64, heads=2, bt=16, dim=64, code=nh.KV8_E4M3):
    return nh.Kv8Cache.empty(blocks, heads, bt, dim, code, device="cpu")


def decode_size(cache, batch=1, heads=8, ctx=1000, window=0):
    return nh.kv8_decode_workspace_size(cache, batch, heads, ctx, window)


def prefill_size(cache, batch=1, heads=8, rows=10, max_rows=10, ctx=1000, window=0):
    return nh.kv8_prefill_workspace_size(cache, batch, heads, rows, max_rows, ctx, window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,q_heads", [(1, 1), (2, 8), (8, 32), (4, 128), (1024, 1024)])
@pytest.mark.parametrize("batch", [1, 3, 64, 65, 1024, 1025, 100000])
def test_workspaces_hold_the_partials_of_a_launch(batch, heads, q_heads, dim):
    cache = cache_of(1, heads, 16, dim)
    for ctx in (1, 256, 257, 5000, 1 << 20, (1 << 31) - 1):
        n = decode_size(cache, batch, q_heads, ctx)
        segments = min(batch, 1024) * heads * -(-q_heads // heads // 16)
        if segments <= 64 and ctx <= 256:
            assert n == 0  # nothing to join
        else:  # 16 rows of values, a maximum and a sum each, at most two per workgroup of 2048
            assert n == 0 and segments <= 64 or COUNTERS < n <= COUNTERS + 4096 * 16 * (dim * 4 + 8)
        n = prefill_size(cache, batch, q_heads, 2 * batch, 2, ctx)
        # tiles of 128 pairs, at most three per CU
        assert n == 0 or COUNTERS < n <= COUNTERS + 3 * 512 * 128 * (dim * 4 + 16)


def test_workspaces_go_by_the_window():
    cache = cache_of()
    assert decode_size(cache, ctx=1 << 20, window=100) <= decode_size(cache, ctx=1 << 20)
    assert decode_size(cache, ctx=1 << 20, window=100) == decode_size(cache, ctx=1 << 14, window=100)
    assert prefill_size(cache, ctx=1 << 20, window=100) == 0 < prefill_size(cache, ctx=1 << 20)


def refusal(call, code, word):
    assert call() == 0
    assert word in nh.last_error(), nh.last_error()
    with pytest.raises(nh.NyionError):
        nh.check(code, "")


@pytest.mark.parametrize("size", [decode_size, prefill_size])
def test_sizes_refuse_what_the_calls_refuse(size):
    assert nh.load().nyion_kv8_decode_workspace_size(None, 1, 1, 1, 0) == 0 and "null" in nh.last_error()
    refusal(lambda: size(cache_of(bt=8)), nh.ERR_UNSUPPORTED, "block_tokens")
    refusal(lambda: size(cache_of(bt=48)), nh.ERR_UNSUPPORTED, "block_tokens")
    refusal(lambda: size(cache_of(bt=512)), nh.ERR_UNSUPPORTED, "block_tokens")
    refusal(lambda: size(cache_of(dim=96)), nh.ERR_UNSUPPORTED, "head_dim")
    refusal(lambda: size(cache_of(code=2)), nh.ERR_INVALID, "code")
    refusal(lambda: size(cache_of(1, 1025)), nh.ERR_UNSUPPORTED, "n_kv_heads")
    refusal(lambda: size(cache_of(), heads=7), nh.ERR_INVALID, "multiple")
    refusal(lambda: size(cache_of(), heads=0), nh.ERR_INVALID, "positive")
    refusal(lambda: size(cache_of(), batch=0), nh.ERR_INVALID, "positive")
    refusal(lambda: size(cache_of(), ctx=0), nh.ERR_INVALID, "positive")
    refusal(lambda: prefill_size(cache_of(), rows=-1), nh.ERR_INVALID, "negative")
    refusal(lambda: prefill_size(cache_of(), rows=1 << 26), nh.ERR_UNSUPPORTED, "2^27")
    refusal(lambda: prefill_size(cache_of(), max_rows=0), nh.ERR_INVALID, "positive")
    refusal(lambda: decode_size(cache_of(1, 1), heads=16385), nh.ERR_UNSUPPORTED, "n_heads")
    odd = cache_of()
    odd.struct.reserved = 1
    refusal(lambda: size(odd), nh.ERR_INVALID, "reserved")
    odd.struct.reserved, odd.struct.k_codes = 0, odd.struct.k_codes + 8
    refusal(lambda: size(odd), nh.ERR_INVALID, "aligned")


def test_structs_are_as_the_header_declares_them():
    assert C.sizeof(nh.Kv8CacheStruct) == 4 * 8 + 6 * 4
    assert C.sizeof(nh.ScoreOptionsStruct) == 4 * 4 + 2 * 8


def test_handles_check_their_tensors():
    k = torch.zeros(3, 2, 16, 64, dtype=torch.uint8)
    s = torch.zeros(3, 2)
    nh.Kv8Cache(k, k.clone(), s, s.clone())
    nh.Kv8Cache(k.view(torch.int8), k.view(torch.int8), s, s, nh.KV8_INT8)
    for bad in ((k.float(), k, s, s), (k, k[:2], s, s), (k[0], k[0], s, s), (k, k, s[:2], s), (k, k, s, s.double()),
                (k.transpose(1, 2).contiguous().transpose(1, 2), k, s, s), (k, k, s.t().contiguous().t(), s)):
        with pytest.raises(nh.NyionError) as e:
            nh.Kv8Cache(*bad)
        assert e.value.code == nh.ERR_INVALID
    for bad in (dict(slopes=torch.zeros(8, dtype=torch.float64)), dict(slopes=torch.zeros(16)[::2]),
                dict(prefix_lens=torch.zeros(8)), dict(window=1 << 31), dict(window=(1 << 32) + 5)):
        with pytest.raises(nh.NyionError) as e:
            nh.ScoreOptions(**bad)
        assert e.value.code == nh.ERR_INVALID


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a device")
def test_without_a_device_the_calls_say_so():
    L, cache, p = nh.load(), cache_of(), 4096
    for call in (lambda: L.nyion_batch_map(p, p, 1, p, 1, 16, 64, p, 4, p, p, p, p, 1, p, None),
                 lambda: L.nyion_kv8_write(cache.ref, p, 1, p, 128, p, 128, nh.IO_F32, None),
                 lambda: L.nyion_kv8_decode_attention(cache.ref, p, 4, p, 1, 64, p, 512, p, 8, nh.IO_F32, None, None,
                                                      0, None),
                 lambda: L.nyion_kv8_prefill_attention_bf16(cache.ref, p, 4, p, p, 1, 1, 1, 64, p, 512, p, 8, None,
                                                            None, 0, None)):
        assert call() == nh.ERR_NO_DEVICE and "device" in nh.last_error()
