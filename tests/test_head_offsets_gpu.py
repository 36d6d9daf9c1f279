"""A head's operators on operands whose rows lie further apart than 32 bits count, in elements."""
from __future__ import annotations

import numpy as np
import pytest

import head_reference as H
from head_reference import BF16, E4M3, F32, I32, Window, close
from helpers import rng
from linalg_hip import backend as B
from test_head_gpu import TOL, logits

pytestmark = pytest.mark.gpu

FAR = (1 << 32) + 40  # elements from one row to the next


class Spread:
    """An [R, C] operand with a pitch of FAR elements, moved row by row."""

    def __init__(self, hb, dtype, data=None, shape=None):
        self.hb, self.dtype = hb, dtype
        shape = list(data.shape if data is not None else shape)
        whole = hb.alloc(dtype, [(shape[0] - 1) * FAR + shape[1]])
        self.t = B.Tensor(whole.storage, dtype, shape, [FAR, 1])
        if data is not None:
            for i, row in enumerate(data):
                whole.storage.buffer.write(np.ascontiguousarray(row), i * FAR * dtype.size_of())

    def read(self):
        buf, size = self.t.storage.buffer, self.dtype.size_of()
        return np.stack([buf.read(H.STORED[self.dtype], i * FAR * size, self.t.shape[1]) for i in range(self.t.shape[0])])


@pytest.fixture()
def hb():
    backend = B.HipBackend(0)
    yield backend
    backend.close()


def test_logits_far_apart(hb):
    g = rng(2100)
    bits = logits(g, 3, 3001, BF16, masks=False)
    x, dx = Spread(hb, BF16, bits), Spread(hb, BF16, shape=[3, 3001])
    tokens = np.array([5, 3000, 17], np.int32)
    tok, lp, h, st = Window(hb, I32, tokens), Window(hb, F32, shape=[3]), Window(hb, F32, shape=[3]), Window(hb, F32, shape=[3, 2])
    top, ids = Window(hb, F32, shape=[3, 9]), Window(hb, I32, shape=[3, 9])
    hb.token_logprobs(x.t, tok.t, 1.0, lp.t, h.t, st.t, top.t, ids.t)
    num = H.values(bits, BF16)
    want = H.logprobs(num, tokens, 9, 1.0)
    close(lp.read(), want[0], TOL, 1e-6, "logprobs")
    assert np.array_equal(ids.read(), want[4])
    one = Window(hb, F32, np.ones(3, np.float32))
    hb.token_logprobs_backward(x.t, tok.t, 1.0, st.t, h.t, one.t, None, dx.t)
    close(H.values(dx.read(), BF16), H.logprobs_backward(num, tokens, 1.0, np.ones(3), np.zeros(3)), 1e-5, 1.01 * H.ROUNDING[BF16], "dlogits")
    losses = Window(hb, F32, shape=[3])
    hb.distill_grad(x.t, ids.t, top.t, None, 1.0, True, losses.t, dx.t)
    loss, grad = H.distill(num, want[4], top.read(), np.ones(3), 1.0, True)
    close(losses.read(), loss, 5e-5, 1e-5, "losses")
    close(H.values(dx.read(), BF16), grad, 2e-5, 1.01 * H.ROUNDING[BF16], "dlogits")


def test_blocks_far_apart(hb):
    g = rng(2200)
    a, b = g.standard_normal((3, 300)).astype(np.float32), g.standard_normal((2, 300)).astype(np.float32)
    x, qa, qb = Spread(hb, BF16, H.to_bits(a, BF16)), Spread(hb, E4M3, shape=[3, 300]), Spread(hb, E4M3, shape=[2, 300])
    sa, sb = Window(hb, F32, shape=[3, 3]), Window(hb, F32, shape=[1, 3])
    hb.quantize_blocks(x.t, qa.t, sa.t)
    hb.quantize_blocks(Window(hb, F32, b).t, qb.t, sb.t)
    wa, wsa = H.quantize(H.values(H.to_bits(a, BF16), BF16).astype(np.float32), 1, F32)
    wb, wsb = H.quantize(b, 128, F32)
    assert np.array_equal(qa.read(), wa) and np.array_equal(qb.read(), wb) and np.array_equal(sa.read(), wsa)
    c = Spread(hb, F32, shape=[3, 2])
    hb.gemm_blocks(qa.t, sa.t, B.transpose_matrix(qb.t), sb.t, c.t)
    va, vb = H.unquantized(wa, wsa, 1, F32), H.unquantized(wb, wsb, 128, F32)
    close(c.read(), va @ vb.T, 140 * 2.0 ** -24 * (np.abs(va) @ np.abs(vb).T), 1e-7, "c")


def test_columns_beyond_one_launch(hb):
    """A's rows far apart, and more rows of B than one launch takes then."""
    g = rng(2300)
    n, k = (1 << 16) + 300, 130
    a, b = g.standard_normal((3, k)).astype(np.float32), g.standard_normal((n, k)).astype(np.float32)
    for block in (1, 128):
        wa, wsa = H.quantize(a, 1, F32)
        wb, wsb = H.quantize(b, block, F32)
        qa, qb, c = Spread(hb, E4M3, wa), Window(hb, E4M3, wb), Window(hb, F32, shape=[3, n], pad=1)
        hb.gemm_blocks(qa.t, Window(hb, F32, wsa).t, B.transpose_matrix(qb.t), Window(hb, F32, wsb).t, c.t)
        va, vb = H.unquantized(wa, wsa, 1, F32), H.unquantized(wb, wsb, block, F32)
        close(c.read(), va @ vb.T, 140 * 2.0 ** -24 * (np.abs(va) @ np.abs(vb).T), 1e-7, "c")
