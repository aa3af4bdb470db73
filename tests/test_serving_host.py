"""The serving calls' argument checks, through the C ABI without a GPU: every check comes
before the device is looked for, so a refused call never reaches one."""
import ctypes

import pytest

from mini_tensorrt_b200 import _lib

A = 0x10000  # a 16-byte aligned address; never read


def prompt(**over):
    a = _lib.AttentionArgs()
    base = dict(q=A, k=A, v=A, out=A, q_row=192, q_head=16, k_row=192, k_head=16, v_row=192, v_head=16, out_row=64,
                out_head=16, rows=5, batch=2, heads=4, kv_heads=2, head_dim=16, x_dtype=_lib.DTYPE_F32,
                dtype=_lib.DTYPE_F32, scale=0.25, cu_rows=A)
    base.update(over)
    for k, v in base.items():
        setattr(a, k, v)
    return a


def paged(**over):
    base = dict(k_pages=A, v_pages=A, page_stride=2 * 16 * 16, num_pages=9, page_size=16, table=A, table_ld=4,
                table_width=4, kv_len=A)
    base.update(over)
    return prompt(**base)


def refuse(fn, a, status):
    assert fn(ctypes.byref(a), None, 0, None) == status
    assert _lib.last_error()
    if status in (_lib.ERR_INVALID_ARG, _lib.ERR_ALIGNMENT):
        assert _lib.lib().mtrtq_attention_workspace_bytes(ctypes.byref(a)) == -1


@pytest.mark.parametrize("over", [
    {"q": None}, {"out": None}, {"cu_rows": None}, {"k": None}, {"v": None}, {"rows": -1}, {"batch": 0},
    {"batch": _lib.MAX_BATCH + 1}, {"heads": 3}, {"heads": 0}, {"kv_heads": 0}, {"heads": 258, "kv_heads": 2},
    {"head_dim": 12}, {"head_dim": 0}, {"head_dim": 136}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
    {"scale": float("inf")}, {"x_dtype": 2}, {"dtype": 7}, {"x_dtype": _lib.DTYPE_BF16}, {"q_row": -16},
    {"out_row": 0}])
def test_prompt_arguments_refused(over):
    refuse(_lib.lib().mtrtq_prompt_attention, prompt(**over), _lib.ERR_INVALID_ARG)


@pytest.mark.parametrize("over", [{"q": A + 4}, {"k": A + 8}, {"q_row": 191}, {"out_head": 6}, {"v_row": 193}])
def test_prompt_alignment_refused(over):
    refuse(_lib.lib().mtrtq_prompt_attention, prompt(**over), _lib.ERR_ALIGNMENT)


@pytest.mark.parametrize("over", [
    {"k_pages": None}, {"v_pages": None}, {"table": None}, {"kv_len": None}, {"k": None}, {"page_size": 8},
    {"page_size": 48}, {"num_pages": 0}, {"table_width": 0}, {"table_ld": 3}, {"page_stride": 511},
    {"table_width": 1 << 28, "table_ld": 1 << 28}])
def test_paged_arguments_refused(over):
    a = paged(**over)
    assert _lib.lib().mtrtq_paged_attention(ctypes.byref(a), None, 0, None) == _lib.ERR_INVALID_ARG
    assert _lib.last_error()


@pytest.mark.parametrize("over", [{"k_pages": A + 4}, {"page_stride": 514}])
def test_paged_alignment_refused(over):
    refuse(_lib.lib().mtrtq_paged_attention, paged(**over), _lib.ERR_ALIGNMENT)


def test_null_arguments_refused():
    lib = _lib.lib()
    assert lib.mtrtq_prompt_attention(None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.mtrtq_paged_attention(None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.mtrtq_attention_workspace_bytes(None) == -1


def select(**over):
    d = dict(logits=A, ldl=100, scores=A, done=A, eos=3, requests=2, beams=4, vocab=100, out_scores=A, parent=A,
             token=A, out_done=A, ws=None, ws_bytes=0)
    d.update(over)
    return _lib.lib().mtrtq_beam_select(*d.values(), None)


@pytest.mark.parametrize("over", [
    {"logits": None}, {"scores": None}, {"done": None}, {"out_scores": None}, {"parent": None}, {"token": None},
    {"out_done": None}, {"ldl": 99}, {"eos": 100}, {"eos": -2}, {"requests": 0}, {"requests": 65536}, {"beams": 0},
    {"beams": _lib.MAX_BEAMS + 1}, {"vocab": 0}, {"vocab": 1 << 29, "ldl": 1 << 29}])
def test_beam_select_arguments_refused(over):
    assert select(**over) == _lib.ERR_INVALID_ARG
    assert _lib.last_error()


def test_beam_workspace_bytes():
    lib = _lib.lib()
    assert lib.mtrtq_beam_workspace_bytes(2, 4, 100) > 0
    assert lib.mtrtq_beam_workspace_bytes(2, 33, 100) == -1
    assert lib.mtrtq_beam_workspace_bytes(0, 4, 100) == -1


def reorder(**over):
    d = dict(parent=A, requests=2, beams=4, table=A, table_ld=5, owned=A, owned_ld=5, width=5, kv_len=A, k_pages=A,
             v_pages=A, layers=2, layer_stride=9 * 512, page_stride=512, num_pages=9, kv_heads=2, page_size=16,
             head_dim=16, dtype=_lib.DTYPE_F32)
    d.update(over)
    return _lib.lib().mtrtq_beam_reorder(*d.values(), None)


@pytest.mark.parametrize("over", [
    {"parent": None}, {"table": None}, {"owned": None}, {"kv_len": None}, {"k_pages": None}, {"v_pages": None},
    {"requests": 0}, {"beams": 0}, {"beams": 33}, {"table_ld": 4}, {"owned_ld": 4}, {"width": 0}, {"layers": 0},
    {"layer_stride": 511}, {"page_stride": 511}, {"num_pages": 0}, {"kv_heads": 0}, {"page_size": 24},
    {"head_dim": 20}, {"dtype": 3}])
def test_beam_reorder_arguments_refused(over):
    assert reorder(**over) == _lib.ERR_INVALID_ARG
    assert _lib.last_error()


@pytest.mark.parametrize("over", [{"k_pages": A + 8}, {"page_stride": 513}, {"layer_stride": 9 * 512 + 2}])
def test_beam_reorder_alignment_refused(over):
    assert reorder(**over) == _lib.ERR_ALIGNMENT
