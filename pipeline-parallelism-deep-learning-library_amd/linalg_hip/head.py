"""A language model's head on 8-bit operands: a teacher that answers with its likeliest
alternatives, and a student that learns from them.

What the last stage of a pipeline does with the backend's head operators, on buffers made once:

* `TeacherHead`: hidden states -> quantize_blocks -> gemm_blocks with weights quantized once ->
  token_logprobs: ids and log probabilities of the k likeliest tokens of each row.
* `StudentHead`: hidden states -> logits by the same product of master weights quantized anew
  after each update -> distill_grad over the logits in place -> both gradients by gemm_blocks on
  operands quantized along the sum (rows of dlogits and the weights' transpose for the hidden
  states, both operands' transposes for the weights) -> sgd_step.

`python -m linalg_hip.head` trains a small student for a few steps and prints the losses.
"""
from __future__ import annotations

from typing import Optional, Tuple

import numpy as np

from .backend import BackendError, DType, HipBackend, Tensor, scales_shape, transpose_matrix


class Quantized:
    """Buffers for the 8-bit form of [rows, cols] matrices, with a scale for each 128 columns and
    `block_rows` (1 or 128) rows."""

    def __init__(self, hb: HipBackend, rows: int, cols: int, block_rows: int, scales: DType = DType.E8M0):
        self.hb = hb
        # Rows of whole 16 bytes are what the product copies straight into LDS.
        pitch = -(-cols // 16) * 16
        stored = hb.alloc(DType.E4M3, [rows, pitch])
        self.q = Tensor(stored.storage, DType.E4M3, [rows, cols], [pitch, 1])
        self.scales = hb.alloc(scales, scales_shape([rows, cols], block_rows))

    def of(self, x: Tensor) -> "Quantized":
        """Holds x's elements from here on (x or a `transpose_matrix` view, of this shape)."""
        self.hb.quantize_blocks(x, self.q, self.scales)
        return self


def product(hb: HipBackend, a: Quantized, b: Quantized, c: Tensor, beta: float = 0.0) -> None:
    """c = a . b^T + beta * c; both operands have the sum along their columns."""
    hb.gemm_blocks(a.q, a.scales, transpose_matrix(b.q), b.scales, c, 1.0, beta)


class TeacherHead:
    """weights [vocab, width] (F32, F16 or BF16), quantized once; calls take `rows` hidden states."""

    def __init__(self, hb: HipBackend, weights: Tensor, rows: int, top: int):
        vocab, width = weights.shape
        self.hb = hb
        self.w = Quantized(hb, vocab, width, 128).of(weights)
        self.x = Quantized(hb, rows, width, 1)
        self.logits = hb.alloc(DType.BF16, [rows, vocab])
        self.ids = hb.alloc(DType.I32, [rows, top])
        self.logprobs = hb.alloc(DType.F32, [rows, top])

    def answer(self, hidden: Tensor, temperature: float = 1.0) -> Tuple[Tensor, Tensor]:
        """(ids, log probabilities) of each row's likeliest tokens; the same buffers every time."""
        product(self.hb, self.x.of(hidden), self.w, self.logits)
        self.hb.token_logprobs(self.logits, temperature=temperature, top_logprobs=self.logprobs, top_ids=self.ids)
        return self.ids, self.logprobs


class StudentHead:
    """Master weights [vocab, width] in F32, trained in place; steps take `rows` hidden states."""

    def __init__(self, hb: HipBackend, weights: Tensor, rows: int):
        if weights.dtype is not DType.F32:
            raise BackendError("Dtype", "master weights are F32")
        vocab, width = weights.shape
        self.hb, self.weights = hb, weights
        self.w = Quantized(hb, vocab, width, 128)    # for the logits
        self.wt = Quantized(hb, width, vocab, 128)   # for the hidden states' gradient
        self.x = Quantized(hb, rows, width, 1)
        self.xt = Quantized(hb, width, rows, 1)      # for the weights' gradient
        self.g = Quantized(hb, rows, vocab, 1)
        self.gt = Quantized(hb, vocab, rows, 1)
        self.logits = hb.alloc(DType.BF16, [rows, vocab])  # and their gradient
        self.losses = hb.alloc(DType.F32, [rows])
        self.dw = hb.alloc(DType.F32, [vocab, width])

    def step(self, hidden: Tensor, ids: Tensor, logprobs: Tensor, weights: Optional[Tensor], temperature: float,
             lr: float, dhidden: Tensor) -> Tensor:
        """One update from a teacher's answers; dhidden = the gradient of the weighted losses with
        respect to the hidden states. Returns the rows' losses."""
        hb = self.hb
        product(hb, self.x.of(hidden), self.w.of(self.weights), self.logits)
        hb.distill_grad(self.logits, ids, logprobs, weights, temperature, True, self.losses, self.logits)
        product(hb, self.g.of(self.logits), self.wt.of(transpose_matrix(self.weights)), dhidden)
        product(hb, self.gt.of(transpose_matrix(self.logits)), self.xt.of(transpose_matrix(hidden)), self.dw)
        hb.sgd_step(self.weights, self.dw, lr)
        return self.losses


def main(rows: int = 256, width: int = 512, vocab: int = 8000, top: int = 32, steps: int = 10) -> list:
    g = np.random.default_rng(0)
    hb = HipBackend(0)
    try:
        def normal(*shape):
            return hb.upload_f32(list(shape), g.standard_normal(shape, dtype=np.float32))
        teacher = TeacherHead(hb, hb.upload_f32([vocab, width], g.standard_normal((vocab, width), dtype=np.float32) / np.sqrt(width) * 3), rows, top)
        student = StudentHead(hb, hb.upload_f32([vocab, width], g.standard_normal((vocab, width), dtype=np.float32) * 0.02), rows)
        hidden, dhidden = normal(rows, width), hb.alloc(DType.F32, [rows, width])
        means = []
        for i in range(steps):
            ids, logprobs = teacher.answer(hidden, 2.0)
            losses = student.step(hidden, ids, logprobs, None, 2.0, 0.02, dhidden)
            means.append(float(hb.download_f32(losses).mean()))
            print(f"step {i}: loss {means[-1]:.4f}", flush=True)
        return means
    finally:
        hb.close()


if __name__ == "__main__":
    main()
