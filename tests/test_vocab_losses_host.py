"""Vocabulary losses without a GPU: a null context is refused at every entry point, the binding's structure has the header's
layout, and the head's f32 form has no pitch."""
import ctypes as C
import os
import re

import pytest

from t0_gpu_b200 import OUT_BF16, OUT_F32, ops
from t0_gpu_b200._lib import LinearLossC, lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_null_context_is_refused():
    L, d = lib(), LinearLossC(rows=1, dim=8, vocab=8)
    assert L.t0b_linear_loss_scratch_bytes(None, C.byref(d), 0) == 0
    assert L.t0b_linear_ce(None, C.byref(d), 0, 0) == -1
    assert L.t0b_linear_topk_distill(None, C.byref(d), 0, 0, 1, 1, 1.0, 0) == -1
    assert L.t0b_topk_distill(None, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1, 1, 1, 1.0, 1.0, 0) == -1


def test_the_structure_follows_the_header():
    with open(os.path.join(ROOT, "include", "t0b200.h")) as f:
        body = re.search(r"typedef struct t0b_linear_loss \{(.*?)\} t0b_linear_loss;", f.read(), re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = [(kind, name.strip()) for kind, names in re.findall(r"(uint64_t|uint32_t|int32_t|float)\s+([^;]+);", body) for name in names.split(",")]
    kinds = {"uint64_t": C.c_uint64, "uint32_t": C.c_uint32, "int32_t": C.c_int32, "float": C.c_float}
    assert [(n, kinds[k]) for k, n in fields] == list(LinearLossC._fields_)


def test_no_word_and_the_limits_are_the_headers():
    with open(os.path.join(ROOT, "include", "t0b200.h")) as f:
        text = f.read()
    assert int(re.search(r"#define T0B_NO_WORD (0x[0-9a-f]+)u", text).group(1), 16) == ops.NO_WORD
    assert re.search(r"#define T0B_MAX_TOPK 1024\b", text)


@pytest.mark.parametrize("w_dtype,ldw", [(OUT_F32, 40), (7, None)])
def test_the_heads_type_and_pitch_are_checked_before_the_call(w_dtype, ldw):
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(None, 16, 16, 16, 4, 8, 32, x_dtype=OUT_BF16, w_dtype=w_dtype, ldw=ldw)
