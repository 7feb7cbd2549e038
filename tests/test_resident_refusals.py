"""What the operators on a caller's tensors refuse before they launch anything (no GPU is needed: no address is read)."""
import ctypes as C

import pytest

from superslm_b200 import abi, build

BAD, OFF = abi.ST["SSLM_INVALID_ARGUMENT"], abi.ST["SSLM_MISALIGNED_BUFFER"]


@pytest.fixture(scope="module")
def dll():
    import os
    return C.CDLL(build.LIB if os.path.exists(build.LIB) else build.build())


def attention(**change):
    a = abi.PrefixAttentionArgs(struct_size=C.sizeof(abi.PrefixAttentionArgs), rows=4, groups=2, heads=12, kv_heads=2, head_dim=128, max_prefix=64, max_suffix=32,
                                q=1 << 20, q_stride=1536, consts=1 << 20, kv=1 << 20, num_pages=100, group_start=1 << 20, prefix_len=1 << 20, prefix_pages=1 << 20,
                                prefix_stride=4, suffix_len=1 << 20, suffix_pages=1 << 20, suffix_stride=2, out=1 << 20, out_stride=1536, row_status=1 << 20)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def pick(**change):
    a = abi.PickArgs(struct_size=C.sizeof(abi.PickArgs), rows=4, vocab=100, num_masks=3, max_history=8, max_bias=8, logits=1 << 20, logits_stride=100,
                     params=1 << 20, history=1 << 20, history_stride=8, history_len=1 << 20, bias_tokens=1 << 20, bias_values=1 << 20, bias_stride=8, bias_len=1 << 20,
                     masks=1 << 20, mask_stride=13, mask_page=1 << 20, out_tokens=1 << 20, out_best=1 << 20, out_logits=1 << 20, out_stride=100)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,want", [
    (dict(struct_size=8), BAD), (dict(rows=-1), BAD), (dict(groups=-1), BAD), (dict(heads=13), BAD), (dict(heads=18), BAD), (dict(kv_heads=0), BAD),
    (dict(heads=0), BAD), (dict(head_dim=96), BAD), (dict(head_dim=0), BAD), (dict(max_prefix=-1), BAD), (dict(max_prefix=32769, prefix_stride=4000), BAD),
    (dict(max_suffix=40000, suffix_stride=4000), BAD), (dict(max_prefix=65), BAD), (dict(max_suffix=33), BAD), (dict(q_stride=1535), BAD), (dict(out_stride=1532), BAD),
    (dict(num_pages=-1), BAD), (dict(num_pages=1 << 40), BAD), (dict(q=None), BAD), (dict(consts=None), BAD), (dict(kv=None), BAD), (dict(group_start=None), BAD),
    (dict(prefix_len=None), BAD), (dict(prefix_pages=None), BAD), (dict(suffix_len=None), BAD), (dict(suffix_pages=None), BAD), (dict(out=None), BAD),
    (dict(out_codes=1 << 20, row_status=None), BAD), (dict(reserved=1), BAD), (dict(rows=65536), BAD), (dict(groups=65536), BAD),
    (dict(kv=(1 << 20) + 8), OFF), (dict(q=(1 << 20) + 1), OFF), (dict(q_stride=1538), OFF), (dict(out=(1 << 20) + 4), OFF), (dict(out_stride=1538), OFF),
    (dict(consts=(1 << 20) + 4), OFF), (dict(fold=(1 << 20) + 2), OFF), (dict(row_status=(1 << 20) + 2), OFF), (dict(out_scales=(1 << 20) + 4), OFF),
    (dict(out_codes=(1 << 20) + 2), OFF), (dict(suffix_pages=(1 << 20) + 2), OFF)])
def test_attention(dll, change, want):
    a = attention(**change)
    assert dll.sslm_b200_attention_prefix_resident(C.byref(a), None) == want


@pytest.mark.parametrize("change,want", [
    (dict(struct_size=8), BAD), (dict(rows=-1), BAD), (dict(rows=65536), BAD), (dict(vocab=0), BAD), (dict(vocab=(1 << 30) + 1, logits_stride=1 << 31), BAD),
    (dict(num_masks=-1), BAD), (dict(logits=None), BAD), (dict(logits_stride=99), BAD), (dict(out_stride=99), BAD), (dict(history_len=None), BAD),
    (dict(max_history=9), BAD), (dict(max_history=-1), BAD), (dict(max_history=65536, history_stride=65536), BAD), (dict(bias_values=None), BAD), (dict(bias_len=None), BAD),
    (dict(max_bias=9), BAD), (dict(max_bias=-1), BAD), (dict(max_bias=1025, bias_stride=1025), BAD), (dict(masks=None), BAD), (dict(mask_stride=12), BAD),
    (dict(out_tokens=None, out_best=None, out_logits=None), BAD), (dict(reserved=1), BAD),
    (dict(logits=(1 << 20) + 2), OFF), (dict(history=(1 << 20) + 1), OFF), (dict(out_logits=(1 << 20) + 2), OFF), (dict(params=(1 << 20) + 2), OFF),
    (dict(mask_page=(1 << 20) + 2), OFF), (dict(out_tokens=(1 << 20) + 2), OFF)])
def test_pick(dll, change, want):
    a = pick(**change)
    assert dll.sslm_b200_pick_resident(C.byref(a), None) == want


def test_no_call(dll):
    assert dll.sslm_b200_attention_prefix_resident(None, None) == BAD and dll.sslm_b200_pick_resident(None, None) == BAD


def test_nothing_to_do(dll):
    for a in (attention(rows=0), attention(groups=0)):
        assert dll.sslm_b200_attention_prefix_resident(C.byref(a), None) == 0
    assert dll.sslm_b200_pick_resident(C.byref(pick(rows=0)), None) == 0


def test_prepared_calls_check_their_tensors():
    torch = pytest.importorskip("torch")
    lib = abi.SslmLib(build.LIB)
    with pytest.raises(ValueError, match="GPU"):
        abi.Pick(lib, logits=torch.zeros((2, 8), dtype=torch.int32), out_tokens=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="logits"):
        abi.Pick(lib, logits=torch.zeros((2, 8)), out_tokens=torch.zeros(2, dtype=torch.int32))


def test_nothing_to_do_on_tensors_without_elements(dll):
    """whose addresses are null"""
    none = {k: None for k in ("logits", "params", "history", "history_len", "bias_tokens", "bias_values", "bias_len", "mask_page", "out_tokens", "out_best", "out_logits")}
    assert dll.sslm_b200_pick_resident(C.byref(pick(rows=0, **none)), None) == 0
    none = {k: None for k in ("q", "consts", "suffix_len", "suffix_pages", "out", "row_status")}
    assert dll.sslm_b200_attention_prefix_resident(C.byref(attention(rows=0, **none)), None) == 0
    assert dll.sslm_b200_pick_resident(C.byref(pick(rows=1, out_tokens=None, out_best=None, out_logits=None)), None) == BAD
