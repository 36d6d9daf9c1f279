"""Refusals of a language model head's operators: their checks run before any device work, in the
order that include/linalg_hip.h gives, and name the first failure (no GPU needed)."""
from __future__ import annotations

import numpy as np
import pytest

import head_reference as H
from head_reference import BF16, E4M3, E8M0, F16, F32, I32
from linalg_hip import backend as B

_next = [1 << 20]


def tensor(dtype, shape, strides=None, offset=0, nbytes=None, base=None):
    """A descriptor whose storage no other has."""
    strides = B.row_major_strides(shape) if strides is None else strides
    need = (offset + sum((n - 1) * s for n, s in zip(shape, strides)) + 1) * H.B.DType(dtype).size_of() if all(shape) else 0
    if base is None:
        base, _next[0] = _next[0], _next[0] + (1 << 32)
    return B.Tensor(B.Storage(base, need if nbytes is None else nbytes), dtype, list(shape), list(strides), offset)


def kind(op, *args):
    with pytest.raises(B.BackendError) as e:
        B.head_checks(op, *args)
    return e.value.kind


PASSED = "UnsupportedDevice"  # every check passes; there is no context


def changed(args, i, t):
    out = list(args)
    out[i] = t
    return out


def test_rows_of_more_columns_than_a_launch_holds():
    for cols, want in ((1 << 29, PASSED), ((1 << 29) + 1, "Shape")):
        wide = [tensor(BF16, [1, cols]), tensor(E4M3, [1, cols]), tensor(F32, [1, -(-cols // 128)])]
        assert kind("quantize_blocks", *wide) == want
        outs = [tensor(F32, [1, 5]), tensor(I32, [1, 5])]
        assert kind("token_logprobs", wide[0], None, 1.0, None, None, None, *outs) == want
        assert kind("token_logprobs", wide[0], None, 1.0, None, tensor(F32, [1]), None, None, None) == PASSED


def test_quantize_blocks_refusals():
    x, q, s = tensor(BF16, [300, 500]), tensor(E4M3, [300, 500]), tensor(F32, [300, 4])
    ok = [x, q, s]
    assert kind("quantize_blocks", *ok) == PASSED
    assert kind("quantize_blocks", *changed(ok, 2, tensor(E8M0, [3, 4]))) == PASSED
    turned = B.transpose_matrix(tensor(F32, [500, 300]))
    assert kind("quantize_blocks", turned, q, s) == PASSED
    for i, t, want in [
            (0, None, "Shape"), (0, tensor(BF16, [300, 499]), "Shape"), (0, tensor(BF16, [300, 500, 1]), "Shape"),
            (2, tensor(F32, [300, 3]), "Shape"), (2, tensor(F32, [4, 4]), "Shape"), (0, tensor(I32, [300, 500]), "Dtype"),
            (1, tensor(F32, [300, 500]), "Dtype"), (2, tensor(F16, [300, 4]), "Dtype"),
            (1, B.transpose_matrix(tensor(E4M3, [500, 300])), "UnsupportedLayout"), (0, tensor(BF16, [300, 500], [499, 1]), "UnsupportedLayout"),
            (0, tensor(BF16, [300, 500], [1000, 2]), "UnsupportedLayout"), (0, tensor(BF16, [300, 500], nbytes=299999), "Shape"),
            (1, tensor(E4M3, [300, 500], base=x.storage.base + 10), "Alias"), (2, tensor(F32, [300, 4], base=q.storage.base), "Alias"),
            (0, tensor(BF16, [300, 500], base=(1 << 50) + 1), "UnsupportedLayout")]:
        assert kind("quantize_blocks", *changed(ok, i, t)) == want, (i, t)
    bad = tensor(BF16, [300, 500])
    bad.dtype = 9
    assert kind("quantize_blocks", bad, q, s) == "Wire"
    assert kind("quantize_blocks", tensor(BF16, [300, 500], base=0), q, s) == "Shape"


def test_gemm_blocks_refusals():
    a, sa, sb, c = tensor(E4M3, [10, 300]), tensor(F32, [10, 3]), tensor(F32, [2, 3]), tensor(BF16, [10, 200])
    b = B.transpose_matrix(tensor(E4M3, [200, 300]))
    ok = [a, sa, b, sb, c, 1.0, 0.0]
    assert kind("gemm_blocks", *ok) == PASSED
    assert kind("gemm_blocks", *changed(ok, 3, tensor(F32, [200, 3]))) == PASSED
    assert kind("gemm_blocks", *changed(ok, 0, tensor(E4M3, [10, 300], [512, 1], 7))) == PASSED
    for i, t, want in [
            (0, tensor(E4M3, [10, 299]), "Shape"), (2, None, "Shape"), (2, tensor(E4M3, [200, 300]), "Shape"),
            (2, tensor(E4M3, [300, 200]), "UnsupportedLayout"), (0, B.transpose_matrix(tensor(E4M3, [300, 10])), "UnsupportedLayout"),
            (4, B.transpose_matrix(tensor(BF16, [200, 10])), "UnsupportedLayout"), (3, tensor(E8M0, [2, 3]), "Dtype"),
            (1, tensor(F32, [10, 2]), "Shape"), (1, tensor(F32, [3, 10]), "Shape"), (0, tensor(F32, [10, 300]), "Dtype"), (4, tensor(E4M3, [10, 200]), "Dtype"),
            (2, B.transpose_matrix(tensor(E4M3, [200, 300], nbytes=59999)), "Shape"), (4, tensor(BF16, [10, 200], base=a.storage.base), "Alias")]:
        assert kind("gemm_blocks", *changed(ok, i, t)) == want, (i, t)
    # Extents and strides that pass what 64 bits hold.
    big = tensor(E4M3, [10, 300], [(1 << 63) - 1, 1], nbytes=1 << 62)
    assert kind("gemm_blocks", *changed(ok, 0, big)) == "Shape"
    assert kind("gemm_blocks", tensor(E4M3, [1 << 31, 300], nbytes=1 << 60), *ok[1:]) == "Shape"


def test_token_logprobs_refusals():
    x, t, lp, h = tensor(BF16, [6, 1000]), tensor(I32, [6]), tensor(F32, [6]), tensor(F32, [6])
    st, top, ids = tensor(F32, [6, 2]), tensor(F32, [6, 128]), tensor(I32, [6, 128])
    ok = [x, t, 1.0, lp, h, st, top, ids]
    assert kind("token_logprobs", *ok) == PASSED
    assert kind("token_logprobs", x, None, 1.0, None, None, None, None, None) == PASSED
    for i, v, want in [
            (0, None, "Shape"), (1, None, "Shape"), (3, None, "Shape"), (6, None, "Shape"), (7, None, "Shape"), (1, tensor(I32, [5]), "Shape"),
            (1, tensor(I32, [6, 1]), "Shape"), (2, 0.0, "Shape"), (2, -1.0, "Shape"), (2, float("nan"), "Shape"), (2, float("inf"), "Shape"),
            (2, 1e-30, "Shape"), (5, tensor(F32, [6, 3]), "Shape"), (6, tensor(F32, [6, 127]), "Shape"), (1, tensor(F32, [6]), "Dtype"),
            (0, tensor(E4M3, [6, 1000]), "Dtype"), (7, tensor(F32, [6, 128]), "Dtype"), (3, tensor(BF16, [6]), "Dtype"),
            (0, B.transpose_matrix(tensor(BF16, [1000, 6])), "UnsupportedLayout"), (1, tensor(I32, [6], [2]), "UnsupportedLayout"),
            (0, tensor(BF16, [6, 1000], offset=8, nbytes=12000), "Shape"), (4, tensor(F32, [6], base=lp.storage.base), "Alias"),
            (6, tensor(F32, [6, 128], base=x.storage.base), "Alias")]:
        assert kind("token_logprobs", *changed(ok, i, v)) == want, (i, v)
    assert kind("token_logprobs", x, t, 1.0, lp, h, st, tensor(F32, [6, 129]), tensor(I32, [6, 129])) == "Shape"


def test_token_logprobs_backward_refusals():
    x, t, st, h = tensor(BF16, [6, 1000]), tensor(I32, [6]), tensor(F32, [6, 2]), tensor(F32, [6])
    g, gh, dx = tensor(F32, [6]), tensor(F32, [6]), tensor(BF16, [6, 1000])
    ok = [x, t, 1.0, st, h, g, gh, dx]
    assert kind("token_logprobs_backward", *ok) == PASSED
    assert kind("token_logprobs_backward", *changed(ok, 7, x)) == PASSED  # in place
    assert kind("token_logprobs_backward", *changed(changed(ok, 4, None), 6, None)) == PASSED
    for i, v, want in [
            (4, None, "Shape"), (5, None, "Shape"), (1, None, "Shape"), (3, None, "Shape"), (7, tensor(BF16, [6, 999]), "Shape"), (2, 0.0, "Shape"),
            (7, tensor(F32, [6, 1000]), "Dtype"), (3, tensor(BF16, [6, 2]), "Dtype"), (7, tensor(BF16, [6, 1000], base=x.storage.base + 2), "Alias"),
            (7, tensor(BF16, [6, 1000], [1001, 1], base=x.storage.base), "Alias"), (5, tensor(F32, [6], base=dx.storage.base), "Alias")]:
        assert kind("token_logprobs_backward", *changed(ok, i, v)) == want, (i, v)


def test_distill_grad_refusals():
    x, ids, v = tensor(F32, [6, 1000]), tensor(I32, [6, 20]), tensor(F32, [6, 20])
    w, losses, dx = tensor(F32, [6]), tensor(F32, [6]), tensor(F32, [6, 1000])
    ok = [x, ids, v, w, 2.0, 1, losses, dx]
    assert kind("distill_grad", *ok) == PASSED
    assert kind("distill_grad", *changed(ok, 7, x)) == PASSED
    assert kind("distill_grad", *changed(changed(ok, 7, None), 3, None)) == PASSED
    for i, t, want in [
            (1, tensor(I32, [6, 19]), "Shape"), (1, None, "Shape"), (6, None, "Shape"), (3, tensor(F32, [5]), "Shape"), (4, 0.0, "Shape"),
            (1, tensor(F32, [6, 20]), "Dtype"), (2, tensor(BF16, [6, 20]), "Dtype"), (7, tensor(BF16, [6, 1000]), "Dtype"),
            (2, tensor(F32, [6, 20], [20, 2], nbytes=1000), "UnsupportedLayout"), (6, tensor(F32, [6], base=x.storage.base), "Alias"),
            (7, tensor(F32, [6, 1000], base=v.storage.base), "Alias")]:
        assert kind("distill_grad", *changed(ok, i, t)) == want, (i, t)
    assert kind("distill_grad", x, tensor(I32, [6, 129]), tensor(F32, [6, 129]), *ok[3:]) == "Shape"


def test_wrong_argument_counts_are_refused():
    with pytest.raises(TypeError):
        B.head_checks("quantize_blocks", tensor(F32, [2, 2]))
    with pytest.raises(B.BackendError):
        B.scales_shape([2, 3], 64)


def test_the_other_operators_refuse_the_new_types():
    x = tensor(E4M3, [4, 4])
    assert B.DType.E4M3.size_of() == 1 and B.DType.I32.size_of() == 4
    with pytest.raises(B.BackendError) as e:
        B.op_checks("gelu", x, tensor(E4M3, [4, 4]))
    assert e.value.kind == "Wire"


def test_the_reference_rounds_to_e4m3():
    """Known values: halfway cases go to even, subnormals have steps of 2^-9, 448 is the largest."""
    x = np.array([0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, 1.0625, 1.1875, 448.0, -432.0, 440.0, np.nan])
    want = [0.0, -0.0, 0.0, 2.0 ** -8, 1.0, 1.25, 448.0, -448.0, 448.0, np.nan]
    got = H.values(H.to_e4m3(x), E4M3)
    assert np.array_equal(got, want, equal_nan=True)
