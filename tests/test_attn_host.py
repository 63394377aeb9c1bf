"""Refusals of the attention operators over buffers (no GPU needed): every bad
argument is turned down before anything touches a device, with its status and
a message that names it."""
import ctypes as C
import subprocess

import pytest

from project_willamette_b200 import _abi
from project_willamette_b200._abi import WLStatus, lib

A = 1 << 20  # an aligned address that nothing follows


def cache(**other):
    return _abi.WlKvPagesI8(**{**dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, page_size=32,
                                      n_kv_heads=5, head_dim=128), **other})


def append(**other):
    return _abi.WlKvAppend(**{**dict(
        q=A, k=A, v=A, q_stride=2560, k_stride=640, v_stride=640, seq_start=A, position=A,
        page_table=A, rope=A, q_out=A, k_out=A, v_out=A, type=0, out_type=1, n_tokens=4, n_seqs=1,
        n_q_heads=20, max_pages=4, n_rot=128, rope_len=64, rope_pairs=0), **other})


def decode(**other):
    return _abi.WlAttnDecode(**{**dict(
        q=A, out=A, q_stride=2560, out_stride=2560, length=A, page_table=A, workspace=A,
        workspace_bytes=1 << 30, type=0, out_type=0, n_seqs=2, n_q_heads=20, max_pages=4, scale=0.1),
        **other})


def prompt(**other):
    return _abi.WlAttnPrompt(**{**dict(
        q=A, k=A, v=A, out=A, q_stride=2560, k_stride=640, v_stride=640, out_stride=2560, seq_start=A,
        type=1, out_type=1, n_tokens=4, n_seqs=1, n_q_heads=20, n_kv_heads=5, head_dim=128, scale=0.1),
        **other})


def refused(rc, status, word):
    assert rc == status
    assert word in lib().wl_last_error().decode()


BAD, TYPE, NOT = WLStatus.INVALID_ARGUMENT, WLStatus.UNSUPPORTED_TENSOR_TYPE, WLStatus.NOT_IMPLEMENTED

CACHE = [
    (dict(page_size=0), BAD, "page_size"), (dict(page_size=48), BAD, "page_size"),
    (dict(page_size=256), BAD, "page_size"), (dict(k=None), BAD, "pages"), (dict(v=A + 8), BAD, "pages"),
    (dict(k_scale=None), BAD, "scales"), (dict(v_scale=A + 2), BAD, "scales"),
    (dict(n_pages=0), BAD, "pages"), (dict(head_dim=96), NOT, "head_dim"),
    (dict(head_dim=256), NOT, "head_dim"), (dict(n_kv_heads=0), BAD, "heads"),
    (dict(n_kv_heads=3), BAD, "heads"),
]


@pytest.mark.parametrize("change,status,word", CACHE)
def test_cache_refusals(change, status, word):
    c = cache(**change)
    refused(lib().wl_dev_rope_kv_append_i8(C.byref(c), C.byref(append()), None), status, word)
    refused(lib().wl_dev_attn_decode_i8(C.byref(c), C.byref(decode()), None), status, word)


@pytest.mark.parametrize("change,status,word", [
    (dict(type=8), TYPE, "8"), (dict(out_type=2), TYPE, "2"), (dict(n_rot=3), BAD, "n_rot"),
    (dict(n_rot=130), BAD, "n_rot"), (dict(rope_pairs=2), BAD, "rope_pairs"),
    (dict(k=None), BAD, "k is NULL"), (dict(v=A + 4), BAD, "v is not 16-byte"),
    (dict(k_stride=636), BAD, "k stride"), (dict(k_stride=642), BAD, "k stride"),
    (dict(q_stride=2559), BAD, "q stride"), (dict(v_stride=1 << 32), BAD, "v stride"),
    (dict(type=1, k_stride=644), BAD, "k stride"), (dict(q=None), BAD, "q_out"),
    (dict(q_out=None), BAD, "q_out"), (dict(k_out=A + 8), BAD, "k_out"), (dict(rope=None), BAD, "rope"),
    (dict(rope=A + 4), BAD, "rope"), (dict(seq_start=None), BAD, "seq_start"),
    (dict(position=A + 2), BAD, "position"), (dict(page_table=None), BAD, "page_table"),
    (dict(max_pages=0), BAD, "max_pages"), (dict(max_pages=1 << 30), BAD, "max_pages"),
    (dict(n_q_heads=21), BAD, "heads"), (dict(n_tokens=1 << 31), BAD, "tokens"),
    (dict(n_seqs=1 << 30), BAD, "sequences"),
])
def test_append_refusals(change, status, word):
    refused(lib().wl_dev_rope_kv_append_i8(C.byref(cache()), C.byref(append(**change)), None), status, word)


@pytest.mark.parametrize("change,status,word", [
    (dict(type=30 + 1), TYPE, "31"), (dict(out_type=14), TYPE, "14"),
    (dict(scale=float("nan")), BAD, "scale"), (dict(scale=float("inf")), BAD, "scale"),
    (dict(q=None), BAD, "q is NULL"), (dict(out=A + 4), BAD, "out is not"),
    (dict(q_stride=2556), BAD, "q stride"), (dict(out_type=1, out_stride=2564), BAD, "out stride"),
    (dict(length=None), BAD, "length"), (dict(page_table=A + 1), BAD, "page_table"),
    (dict(max_pages=0), BAD, "max_pages"), (dict(workspace=None), BAD, "workspace"),
    (dict(workspace=A + 8), BAD, "workspace"), (dict(workspace_bytes=8), BAD, "workspace"),
    (dict(n_seqs=70000), BAD, "sequences"), (dict(n_q_heads=0), BAD, "heads"),
])
def test_decode_refusals(change, status, word):
    refused(lib().wl_dev_attn_decode_i8(C.byref(cache()), C.byref(decode(**change)), None), status, word)


@pytest.mark.parametrize("change,status,word", [
    (dict(type=0), TYPE, "0"), (dict(out_type=30), TYPE, "30"), (dict(type=30, out_type=1), TYPE, "1"),
    (dict(head_dim=80), NOT, "head_dim"), (dict(n_kv_heads=6), BAD, "heads"),
    (dict(scale=float("-inf")), BAD, "scale"), (dict(q=None), BAD, "q is NULL"),
    (dict(k=A + 8), BAD, "k is not"), (dict(k_stride=644), BAD, "k stride"),
    (dict(v_stride=0), BAD, "v stride"), (dict(out_stride=2552), BAD, "out stride"),
    (dict(seq_start=None), BAD, "seq_start"), (dict(n_tokens=1 << 31), BAD, "tokens"),
])
def test_prompt_refusals(change, status, word):
    refused(lib().wl_dev_attn_prompt(C.byref(prompt(**change)), None), status, word)


def test_null_structs_are_refused():
    L = lib()
    refused(L.wl_dev_rope_kv_append_i8(None, C.byref(append()), None), BAD, "cache")
    refused(L.wl_dev_rope_kv_append_i8(C.byref(cache()), None, None), BAD, "args")
    refused(L.wl_dev_attn_decode_i8(None, C.byref(decode()), None), BAD, "cache")
    refused(L.wl_dev_attn_decode_i8(C.byref(cache()), None, None), BAD, "args")
    refused(L.wl_dev_attn_prompt(None, None), BAD, "args")


def test_nothing_to_do_is_no_error():
    """No tokens or sequences: done before the buffers are looked at."""
    L = lib()
    for change in (dict(n_tokens=0, k=None), dict(n_seqs=0, k=None)):
        assert L.wl_dev_rope_kv_append_i8(C.byref(cache()), C.byref(append(**change)), None) == 0
    assert L.wl_dev_attn_decode_i8(C.byref(cache()), C.byref(decode(n_seqs=0, q=None)), None) == 0
    for change in (dict(n_tokens=0, q=None), dict(n_seqs=0, q=None)):
        assert L.wl_dev_attn_prompt(C.byref(prompt(**change)), None) == 0


def test_structs_match_the_header(tmp_path):
    pairs = [("wl_kv_pages_i8", _abi.WlKvPagesI8), ("wl_kv_append", _abi.WlKvAppend),
             ("wl_attn_decode", _abi.WlAttnDecode), ("wl_attn_prompt", _abi.WlAttnPrompt)]
    body = "".join(f'printf("%zu", sizeof({c}));' + "".join(
        f'printf(" %zu", offsetof({c}, {n}));' for n, _ in p._fields_) + 'printf("\\n");' for c, p in pairs)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "willamette_b200.h"\n'
                   "int main(void) {" + body + "return 0; }\n")
    exe = tmp_path / "s"
    import os
    subprocess.run(["gcc", "-std=c11", "-I", os.path.dirname(_abi.HEADER_PATH), str(src), "-o", str(exe)],
                   check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (_, p) in zip(lines, pairs):
        assert [int(x) for x in line.split()] == [C.sizeof(p)] + [getattr(p, n).offset for n, _ in p._fields_]
