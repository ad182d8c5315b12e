"""The C ABI of the 8-bit KV cache on the host (no GPU needed): bad arguments come back as a status
before CUDA is touched."""

from __future__ import annotations

import ctypes

import pytest

import svllm_capi as capi

INVALID, TOO_LARGE, UNSUPPORTED = 1, 2, 3
P = 256  # stands for an aligned pointer; nothing is launched
FREQ = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p)


def norm_write(**change):
    a = dict(q=P, k=P, v=P, q_weight=P, k_weight=P, positions=P, pos_type=1, slot_mapping=P,
             k_cache=P, v_cache=P, k_scale=P, v_scale=P, num_slots=64, num_tokens=3, num_heads=4,
             num_kv_heads=2, head_dim=64, q_row_stride=512, k_row_stride=512, v_row_stride=512,
             eps=1e-6, inv_freq=FREQ, stream=None)
    a.update(change)
    return capi.lib().svllm_qk_norm_rope_cache_fp8_bf16(*a.values())


def write(**change):
    a = dict(q=P, k=P, v=P, positions=P, pos_type=1, slot_mapping=P, k_cache=P, v_cache=P,
             k_scale=P, v_scale=P, num_slots=64, num_tokens=3, num_heads=4, num_kv_heads=2,
             head_dim=64, q_row_stride=512, k_row_stride=512, v_row_stride=512, inv_freq=FREQ,
             stream=None)
    a.update(change)
    return capi.lib().svllm_rope_cache_fp8_bf16(*a.values())


def read(**change):
    a = dict(k_out=P, v_out=P, k_cache=P, v_cache=P, k_scale=P, v_scale=P, num_blocks=4,
             block_size=16, block_tables=P, max_blocks=2, seq_lens=P, num_seqs=1, num_kv_heads=2,
             head_dim=64, stream=None)
    a.update(change)
    return capi.lib().svllm_cache_read_fp8_bf16(*a.values())


def commit(pointer=P, **change):
    one = ctypes.cast((ctypes.c_void_p * 1)(pointer), ctypes.c_void_p)
    a = dict(k_scales=one, v_scales=one, num_layers=1, num_slots=16, num_kv_heads=5, path=P,
             num_accepted=P, slot_mapping=P, query_start_loc=P, num_seqs=1, num_tokens=4,
             max_query_len=8, stream=None)
    a.update(change)
    return capi.lib().svllm_tree_commit_scales(*a.values())


@pytest.mark.parametrize("call, change, status", [
    (norm_write, {"q_weight": None}, INVALID),
    (norm_write, {"k_weight": None}, INVALID),
    (write, {"num_tokens": -1}, INVALID),
    (write, {"num_kv_heads": 0}, INVALID),
    (write, {"num_slots": -1}, INVALID),
    (write, {"pos_type": 2}, INVALID),
    (write, {"inv_freq": None}, INVALID),
    (write, {"q_row_stride": 255}, INVALID),
    (write, {"k_row_stride": 127}, INVALID),
    (write, {"v_row_stride": 127}, INVALID),
    (write, {"q": None}, INVALID),
    (write, {"v": None}, INVALID),
    (write, {"k_scale": None}, INVALID),
    (write, {"slot_mapping": P + 4}, INVALID),
    (write, {"num_heads": 1 << 17, "q_row_stride": 1 << 40}, TOO_LARGE),
    (write, {"head_dim": 32}, UNSUPPORTED),
    (write, {"k_cache": P + 8}, UNSUPPORTED),
    (read, {"num_seqs": -1}, INVALID),
    (read, {"block_size": 0}, INVALID),
    (read, {"num_blocks": 0}, INVALID),
    (read, {"k_out": None}, INVALID),
    (read, {"v_scale": None}, INVALID),
    (read, {"block_tables": None}, INVALID),
    (read, {"num_seqs": 1 << 24, "max_blocks": 1 << 12}, TOO_LARGE),
    (read, {"max_blocks": 1 << 28}, TOO_LARGE),
    (read, {"block_size": 1 << 20}, TOO_LARGE),
    (read, {"head_dim": 96}, UNSUPPORTED),
    (read, {"v_out": P + 8}, UNSUPPORTED),
    (commit, {}, INVALID),  # K and V the same
    (commit, {"num_kv_heads": 0}, INVALID),
    (commit, {"pointer": None}, INVALID),
    (commit, {"max_query_len": 1025}, TOO_LARGE),
], ids=str)
def test_bad_arguments(call, change, status):
    assert call(**change) == status


def test_nothing_to_do_is_ok():
    assert norm_write(num_tokens=0) == 0 and write(num_tokens=0) == 0
    assert read(num_seqs=0) == 0 and read(max_blocks=0) == 0
    assert commit(num_seqs=0) == 0 and commit(num_layers=0) == 0
