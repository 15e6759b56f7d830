"""Limits of the ragged operators that are found before any CUDA call (CPU)."""

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200 import _lib


def test_workspace_alignment():
    lib = _lib.load()
    pool = _lib.KVLayout(k=16, v=16, dtype=2, head_dim=128, batch=2, num_kv_heads=2, stride_h=2048,
                         stride_p=4096, stride_t=128, page_size=16, num_slots=7, page_table=16,
                         pt_stride_b=3, num_tokens=48)
    q, o = _lib.Query(16, 2, 8, 1, 1024, 128, 128), _lib.Output(16, 2, 0, 1024, 128, 128)
    size = lib.rkv_ragged_decode_attention_workspace_size(q, pool)
    for at in (8, 24, 1):
        assert lib.rkv_ragged_decode_attention(q, pool, 16, None, 0.0, o, None, at, size, None) == 5
