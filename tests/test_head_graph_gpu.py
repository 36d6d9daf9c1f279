"""A head's operators under HIP graph capture: kernels only, so a step that is captured once replays on new
inputs, with eager calls on the same context (which use the same scratch) between the replays."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import head_reference as H
from head_reference import BF16, E4M3, E8M0, F32, I32, Window
from helpers import rng
from linalg_hip import _native as N
from linalg_hip import backend as B
from test_graph_gpu import Hip

pytestmark = pytest.mark.gpu


def call(hb, stream, name, *args):
    refs = [ctypes.byref(a.t.to_c()) if isinstance(a, Window) else ctypes.byref(a.to_c()) if isinstance(a, B.Tensor) else a for a in args]
    assert getattr(N.lib(), "lg_backend_" + name)(hb.ctx.handle, stream, *refs) == 0


def test_a_captured_head_replays_like_eager_work():
    hip, hb = Hip(), B.HipBackend(0)
    q = hb.ctx.new_stream()
    try:
        g = rng(2000)
        rows, width, vocab, top = 3, 256, 70001, 20
        x, xq, xs = Window(hb, F32, shape=[rows, width]), Window(hb, E4M3, shape=[rows, width]), Window(hb, E8M0, shape=[rows, 2])
        w, ws = H.quantize(g.standard_normal((vocab, width)).astype(np.float32), 128, E8M0)
        w, ws = Window(hb, E4M3, w), Window(hb, E8M0, ws)
        logits, dlogits = Window(hb, BF16, shape=[rows, vocab]), Window(hb, BF16, shape=[rows, vocab])
        ids, logprobs = Window(hb, I32, shape=[rows, top]), Window(hb, F32, shape=[rows, top])
        entropy, losses = Window(hb, F32, shape=[rows]), Window(hb, F32, shape=[rows])
        outs = [logits, ids, logprobs, entropy, losses, dlogits]

        def step(stream):
            call(hb, stream, "quantize_blocks", x, xq, xs)
            call(hb, stream, "gemm_blocks", xq, xs, B.transpose_matrix(w.t), ws, logits, 1.0, 0.0)
            call(hb, stream, "token_logprobs", logits, None, 1.0, None, entropy, None, logprobs, ids)
            call(hb, stream, "distill_grad", logits, ids, logprobs, None, 2.0, 1, losses, dlogits)

        hb.sync()
        graph, exe = hip.capture(q.handle, lambda: step(q.handle))
        for replay in range(4):
            x.whole.storage.buffer.write(g.standard_normal((rows, width)).astype(np.float32))
            step(None)
            hb.sync()
            want = [o.whole.storage.buffer.read(np.uint8).copy() for o in outs]
            for o in outs:
                o.whole.storage.buffer.write(np.zeros(o.whole.storage.nbytes, np.uint8))
            hb.sync()
            assert hip.h.hipGraphLaunch(exe, q.handle) == 0
            q.wait_until_completed()
            for o, v in zip(outs, want):
                assert np.array_equal(o.whole.storage.buffer.read(np.uint8)[:o.whole.storage.nbytes], v[:o.whole.storage.nbytes]), replay
        hip.h.hipGraphExecDestroy(exe)
        hip.h.hipGraphDestroy(graph)
    finally:
        q.close()
        hb.close()
