"""A teacher's answers and a student's step through linalg_hip.head, against the same step in 64 bits
on the operands as they were quantized (head_reference.py restates the quantization).

The step's products are checked within the products' own bounds (test_head_gpu.py): the logits and the gradient
are bf16, so what is computed from them takes the device's own as its input.
"""
from __future__ import annotations

import numpy as np
import pytest

import head_reference as H
from head_reference import BF16, E8M0, F32, I32, close
from helpers import rng
from linalg_hip import backend as B
from linalg_hip import head

pytestmark = pytest.mark.gpu


def bits(hb, t):
    return np.frombuffer(hb.download(t), H.STORED[t.dtype]).reshape(t.shape)


def product_bound(a, b):
    """Of sums of a @ b.T: f32 sums of up to K terms, or of groups of eight kept to 2^-13 of the largest."""
    return (a.shape[1] + 4) * 2.0 ** -24 * (np.abs(a) @ np.abs(b).T) + 2.0 ** -16 * (np.abs(a) @ np.abs(b).T) / np.sqrt(a.shape[1] / 128)


def as_quantized(x, block):
    q, s = H.quantize(np.ascontiguousarray(x, dtype=np.float32), block, E8M0)
    return H.unquantized(q, s, block, E8M0)


@pytest.mark.parametrize("rows,width,vocab,top", [(48, 256, 1000, 12), (130, 200, 999, 20), (1, 128, 4097, 5)])
def test_a_distillation_step(rows, width, vocab, top):
    g = rng(1900 + rows)
    hb = B.HipBackend(0)
    try:
        x0 = g.standard_normal((rows, width)).astype(np.float32)
        wt = (3 * g.standard_normal((vocab, width)) / np.sqrt(width)).astype(np.float32)
        ws = (0.1 * g.standard_normal((vocab, width))).astype(np.float32)
        hidden, dhidden = hb.upload_f32([rows, width], x0), hb.alloc(F32, [rows, width])
        teacher = head.TeacherHead(hb, hb.upload_f32([vocab, width], wt), rows, top)
        student = head.StudentHead(hb, hb.upload_f32([vocab, width], ws), rows)
        t = 2.0

        ids, logprobs = teacher.answer(hidden, t)
        ids, logprobs = bits(hb, ids).copy(), bits(hb, logprobs).copy()
        xq, wq = as_quantized(x0, 1), as_quantized(wt, 128)
        logits = H.values(bits(hb, teacher.logits), BF16)
        close(logits, xq @ wq.T, product_bound(xq, wq), 1.01 * H.ROUNDING[BF16], "the teacher's logits")
        want = H.logprobs(logits, np.full(rows, -1), top, t)
        assert np.array_equal(ids, want[4])
        close(logprobs, want[3], 1e-5, 1e-6, "the teacher's log probabilities")

        sq = as_quantized(ws, 128)
        losses = hb.download_f32(student.step(hidden, teacher.ids, teacher.logprobs, None, t, 0.5, dhidden))
        # The loss from the exact logits: each is off by half a unit of bf16 and the product's bound.
        off = (product_bound(xq, sq) + H.ROUNDING[BF16] * np.abs(xq @ sq.T)).max(1)
        want_loss, want_grad = H.distill(xq @ sq.T, ids, logprobs, np.ones(rows), t, True)
        close(losses, want_loss, 2 * t * off + 1e-5, 1e-5, "losses")
        grad = H.values(bits(hb, student.logits), BF16)
        close(grad, want_grad, (2 * t * off / t)[:, None] * np.abs(grad).max(1, keepdims=True) + 1e-5, 1.01 * H.ROUNDING[BF16], "dlogits")
        # Both products back, from the gradient as the device has it.
        gq, gtq = as_quantized(grad, 1), as_quantized(grad.T, 1)
        close(bits(hb, dhidden), gq @ as_quantized(ws.T, 128).T, product_bound(gq, as_quantized(ws.T, 128)), 1e-6, "dhidden")
        dw = gtq @ as_quantized(x0.T, 1).T
        close(bits(hb, student.weights), ws - 0.5 * dw, 0.5 * product_bound(gtq, as_quantized(x0.T, 1)) + 2.0 ** -23 * np.abs(ws), 1e-6, "weights")
    finally:
        hb.close()


def test_the_example_learns(capsys):
    losses = head.main(rows=64, width=128, vocab=2000, top=16, steps=6)
    assert all(b < a for a, b in zip(losses, losses[1:])), losses
    assert capsys.readouterr().out.count("loss") == 6


def test_master_weights_are_f32():
    hb = B.HipBackend(0)
    try:
        with pytest.raises(B.BackendError):
            head.StudentHead(hb, hb.alloc(BF16, [8, 8]), 1)
    finally:
        hb.close()
