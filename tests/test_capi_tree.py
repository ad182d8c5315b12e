"""The C ABI of the drafted-tree operators on the host (no GPU needed): bad arguments come back as a
status before CUDA is touched."""

from __future__ import annotations

import ctypes

import pytest

import svllm_capi as capi

INVALID, TOO_LARGE, UNSUPPORTED = 1, 2, 3
P = 256  # stands for an aligned pointer; nothing is launched


def plan(**change):
    a = dict(context_lens=P, query_lens=P, num_seqs=1, block_tables=P, max_blocks=4,
             blocks_owned=P, free_blocks=P, free_capacity=4, free_count=P, block_size=16,
             parents=P, max_query_len=8, num_tokens=4, query_start_loc=P, seq_lens=P,
             slot_mapping=P, positions=P, tree_mask=P, blocks_owned_out=2 * P,
             free_count_out=2 * P, stream=None)
    a.update(change)
    return capi.lib().svllm_paged_plan(*a.values())


def attention(**change):
    a = dict(out=P, q=P, q_token_stride=256, k_cache=P, v_cache=P, num_blocks=4, block_size=16,
             block_tables=P, max_blocks=2, seq_lens=P, query_start_loc=P, num_seqs=1,
             num_tokens=3, num_heads=4, num_kv_heads=2, head_dim=64, tree_mask=P, mask_words=1,
             scale=0.125, workspace=P, workspace_bytes=0, stream=None)
    a.update(change)
    return capi.lib().svllm_tree_attention_bf16(*a.values())


def accept(**change):
    a = dict(ids=P, id_type=1, targets=P, parents=P, query_start_loc=P, seq_lens=P,
             context_lens=P, num_seqs=1, num_tokens=4, max_query_len=8, path=P, tokens=P,
             num_accepted=P, context_lens_out=P, stream=None)
    a.update(change)
    return capi.lib().svllm_tree_accept(*a.values())


def commit(pointer=P, **change):
    one = ctypes.cast((ctypes.c_void_p * 1)(pointer), ctypes.c_void_p)
    a = dict(k_caches=one, v_caches=one, num_layers=1, num_slots=16, row_bytes=64, path=P,
             num_accepted=P, slot_mapping=P, query_start_loc=P, num_seqs=1, num_tokens=4,
             max_query_len=8, stream=None)
    a.update(change)
    return capi.lib().svllm_tree_commit(*a.values())


@pytest.mark.parametrize("call, change, status", [
    (plan, {"num_seqs": -1}, INVALID),
    (plan, {"num_tokens": -1}, INVALID),
    (plan, {"max_blocks": 0}, INVALID),
    (plan, {"block_size": 0}, INVALID),
    (plan, {"max_query_len": 0}, INVALID),
    (plan, {"tree_mask": None}, INVALID),
    (plan, {"query_lens": None}, INVALID),
    (plan, {"slot_mapping": None}, INVALID),
    (plan, {"blocks_owned_out": P}, INVALID),       # the input array
    (plan, {"free_count_out": P}, INVALID),
    (plan, {"max_query_len": 1025}, TOO_LARGE),
    (plan, {"num_tokens": 1 << 31}, TOO_LARGE),
    (plan, {"max_blocks": 1 << 30, "block_size": 4}, TOO_LARGE),
    (attention, {"num_heads": 5}, INVALID),
    (attention, {"num_blocks": 0}, INVALID),
    (attention, {"scale": 0.0}, INVALID),
    (attention, {"scale": float("nan")}, INVALID),
    (attention, {"mask_words": 0}, INVALID),
    (attention, {"q_token_stride": 255}, INVALID),
    (attention, {"q": None}, INVALID),
    (attention, {"head_dim": 96, "q_token_stride": 384}, UNSUPPORTED),
    (attention, {"q_token_stride": 260}, UNSUPPORTED),
    (attention, {"k_cache": P + 8}, UNSUPPORTED),
    (attention, {"mask_words": 17}, TOO_LARGE),
    (attention, {"num_tokens": 1 << 61}, TOO_LARGE),
    (attention, {"num_blocks": 1 << 30}, TOO_LARGE),
    (attention, {"max_blocks": 1 << 28}, TOO_LARGE),
    (accept, {"id_type": 2}, INVALID),
    (accept, {"max_query_len": 0}, INVALID),
    (accept, {"targets": None}, INVALID),
    (accept, {"path": None}, INVALID),
    (accept, {"max_query_len": 1025}, TOO_LARGE),
    (commit, {"row_bytes": 0}, INVALID),
    (commit, {"num_layers": -1}, INVALID),
    (commit, {"pointer": None}, INVALID),
    (commit, {"path": None}, INVALID),
    (commit, {"row_bytes": 40}, UNSUPPORTED),
    (commit, {"pointer": P + 8}, UNSUPPORTED),
    (commit, {"max_query_len": 1025}, TOO_LARGE),
], ids=str)
def test_bad_arguments(call, change, status):
    assert call(**change) == status


def test_a_cache_given_twice():
    assert commit() == INVALID  # K and V the same
    planes = (ctypes.c_void_p * 400)(*(P + 16 * i for i in range(400)))
    for layers in (2, 200):
        at = [ctypes.cast(ctypes.byref(planes, 8 * i), ctypes.c_void_p) for i in (0, layers - 1)]
        assert commit(k_caches=at[0], v_caches=at[1], num_layers=layers) == INVALID


def test_nothing_to_do_is_ok():
    assert attention(num_tokens=0) == 0
    assert accept(num_seqs=0) == 0
    assert commit(num_seqs=0) == 0 and commit(num_layers=0) == 0


def test_workspace_size_refusals():
    size = ctypes.c_int64(0)
    assert capi.lib().svllm_tree_attention_workspace_bytes(96, ctypes.byref(size)) == UNSUPPORTED
    assert capi.lib().svllm_tree_attention_workspace_bytes(64, None) == INVALID
