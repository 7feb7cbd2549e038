"""Compaction in place: the tables may be their own output, row for row (no GPU is needed: no address is read)."""
import ctypes as C

import pytest

from superslm_b200 import abi, build

BAD, AT = abi.ST["SSLM_INVALID_ARGUMENT"], 1 << 20


@pytest.fixture(scope="module")
def dll():
    import os
    return C.CDLL(build.LIB if os.path.exists(build.LIB) else build.build())


@pytest.mark.parametrize("tables_stride,out_stride", [(7, 8), (9, 7), (1 << 33, 7)])
@pytest.mark.parametrize("sequences", [2, 300])
def test_rows_of_tables_in_place_are_their_own(dll, sequences, tables_stride, out_stride):
    """with another stride a sequence's output is another one's input"""
    a = abi.CompactArgs(struct_size=C.sizeof(abi.CompactArgs), sequences=sequences, table_pages=7, planes=3, page_bytes=512, num_pages=50, kv=AT, holders=AT, tables=4 * AT,
                        tables_stride=tables_stride, lengths=AT, out_holders=2 * AT, out_tables=4 * AT, out_stride=out_stride, new_of=AT, moves=AT, counts=AT, status=AT)
    assert dll.sslm_b200_compact_resident(C.byref(a), None) == BAD
