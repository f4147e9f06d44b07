"""Batched operators whose launch would have 2^32 threads or more: refused before anything is launched, without a GPU."""

import ctypes as C

import pytest

from q4llm._lib import LIB
from test_paged_cpu import ERR, F16, FAKE, append, attend, paged, rope


@pytest.mark.parametrize("T", [1 << 24, (1 << 25) + 3, (1 << 31) // 63 - 1])
def test_rope_and_append(T):
    r = rope(rot_dim=1024)
    assert LIB.raw("rope_rotate")(FAKE, 64512, 1024, FAKE, 64512, 1024, F16, T, 63, 1024, FAKE, C.byref(r), 0, None) == ERR["SHAPE"]
    assert append(kv=paged(n_kv=20, head_dim=1024, cu_q=FAKE), T=T, r=r, n_q=23, strides=(1024 * 63, 1024) * 4) == ERR["SHAPE"]


def test_attention():
    # 2^24 workgroups of single tokens; 2^27 rows of which some have several ranges of keys
    assert attend(kv=paged(batch=1 << 24, n_kv=1), T=1 << 24, n_q=1, shared=0) == ERR["SHAPE"]
    many = dict(kv=paged(batch=1, n_kv=1, head_dim=128, max_pages=1 << 10, table_stride=1 << 10, num_pages=1 << 10), T=(1 << 27) + 256, n_q=1,
                L=1 << 14, shared=0, row=128, head=128)
    assert attend(**many) == ERR["SHAPE"]


def test_verification():
    b = (1 << 24)
    assert LIB.raw("spec_verify")(FAKE, 1, None, 0, 0, FAKE, 0, 0, FAKE, 2, None, b, 1, 1, FAKE, FAKE, FAKE, 1 << 40, None) == ERR["SHAPE"]
