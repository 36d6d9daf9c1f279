"""A language model head's operators on the GPU against 64-bit references (head_reference.py).

Bounds, each derived from the operators' arithmetic:
* quantize_blocks: bit for bit; its definition names every rounding.
* gemm_blocks: a block's 128 products are summed in f32 (128 roundings of at most the sum S of
  absolute products), the scaled blocks by one multiply and one multiply-add each, alpha and beta
  add three more: (128 + 2 blocks + 3) * 2^-24 * S, then the rounding to c's type.
* softmax: an exponent d = (x - max) log2(e) / T is off by at most 2^-22 |d| (three roundings and
  that of log2(e) / T), so 2^d by 2^-22 ln 2 |d| and the instruction's 2^-22; weighted by p, |d| is
  at most log2 V + 3 on average: log sums and entropies are within 2^-22 (log2 V + 4), entropies
  within twice that times their own exponents, and results of f32 add 2^-23 of themselves. TOL
  holds that for V up to 2^19: 1e-5; entropies 4e-5.
* gradients: p is off by at most 2^-22 (|d| + 2) with |d| 2^d <= 0.54 max, so 1e-5 of the row's
  largest coefficient, then the rounding to the type.
"""
from __future__ import annotations

import numpy as np
import pytest

import head_reference as H
from head_reference import BF16, E4M3, E8M0, F16, F32, I32, Window, close
from helpers import rng
from linalg_hip import backend as B

pytestmark = pytest.mark.gpu

TOL, TOL_ENTROPY = 1e-5, 4e-5


@pytest.fixture()
def hb():
    backend = B.HipBackend(0)
    yield backend
    backend.close()


# ------------------------------------------------------------------------------- quantize


def matrix(g, r, c, dtype):
    x = g.standard_normal((r, c)) * np.exp(g.standard_normal((r, 1)))
    return H.to_bits(x, dtype)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,pad", [((1, 1), 0), ((1, 128), 0), ((3, 129), 1), ((130, 127), 8), ((257, 640), 0), ((5, 1000), 24), ((128, 8), 0)])
def test_quantize_blocks_bit_for_bit(hb, shape, pad, dtype, block, scales, transposed):
    g = rng(100 + shape[0])
    r, c = shape
    bits = matrix(g, c, r, dtype) if transposed else matrix(g, r, c, dtype)
    x = Window(hb, dtype, bits, pad=pad, offset=3)
    q = Window(hb, E4M3, shape=shape, pad=pad, offset=5)
    s = Window(hb, scales, shape=B.scales_shape(shape, block), pad=1)
    hb.quantize_blocks(B.transpose_matrix(x.t) if transposed else x.t, q.t, s.t)
    num = H.values(bits.T if transposed else bits, dtype).astype(np.float32)
    want_q, want_s = H.quantize(num, block, scales)
    assert np.array_equal(s.read().view(np.uint8), want_s.view(np.uint8))
    assert np.array_equal(q.read(), want_q)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(256, 1024), (128, 128), (1000, 640), (1150, 2304), (2000, 64)])
def test_quantize_blocks_of_whole_lines(hb, shape, dtype, transposed):
    """Operands of their own, whose rows are whole lines of memory or nearly."""
    g = rng(150 + shape[0])
    r, c = shape
    bits = matrix(g, c, r, dtype) if transposed else matrix(g, r, c, dtype)
    for block in (1, 128):
        x, q, s = Window(hb, dtype, bits), Window(hb, E4M3, shape=shape), Window(hb, E8M0, shape=B.scales_shape(shape, block))
        hb.quantize_blocks(B.transpose_matrix(x.t) if transposed else x.t, q.t, s.t)
        want_q, want_s = H.quantize(H.values(bits.T if transposed else bits, dtype).astype(np.float32), block, E8M0)
        assert np.array_equal(s.read(), want_s) and np.array_equal(q.read(), want_q)


@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_blocks_at_the_ends_of_the_range(hb, block, scales):
    """Zeros, subnormals, the largest numbers, every significand beside 448's, infinities and NaN."""
    x = np.zeros((9, 256), np.float32)
    x[1, :3] = [1e-45, -1e-40, 1e-38]
    x[2, :4] = [3.4028235e38, -3.4e38, 1.0, 2.0 ** 100]
    x[3, :128] = np.linspace(-448, 448, 128)
    x[4, 0] = np.nextafter(np.float32(448), np.float32(1000))
    x[5, 7], x[5, 130] = np.inf, 1.5
    x[6, 200], x[6, 3] = np.nan, -2.0
    x[7, :256] = np.exp2(np.arange(256) / 16.0 - 8.0)
    x[8, 0] = -np.inf
    xs, q = Window(hb, F32, x), Window(hb, E4M3, shape=x.shape)
    s = Window(hb, scales, shape=B.scales_shape(x.shape, block))
    hb.quantize_blocks(xs.t, q.t, s.t)
    want_q, want_s = H.quantize(x, block, scales)
    assert np.array_equal(H.values(s.read(), scales), H.values(want_s, scales), equal_nan=True)
    assert np.array_equal(H.values(q.read(), E4M3), H.values(want_q, E4M3), equal_nan=True)


# -------------------------------------------------------------------------------- product


def product(hb, g, m, n, k, scales, ba, bb, out, alpha=1.0, beta=0.0, pad=(0, 0, 0), offset=0, spoil=None):
    xa = (g.standard_normal((m, k)) * np.exp(g.standard_normal((m, 1)))).astype(np.float32)
    xb = g.standard_normal((n, k)).astype(np.float32)
    if spoil is not None:
        spoil(xa, xb)
    qa, sa = H.quantize(xa, ba, scales)
    qb, sb = H.quantize(xb, bb, scales)
    c0 = H.to_bits(g.standard_normal((m, n)), out)
    a, b = Window(hb, E4M3, qa, pad=pad[0], offset=offset), Window(hb, E4M3, qb, pad=pad[1], offset=offset)
    wsa, wsb = Window(hb, scales, sa, pad=pad[2]), Window(hb, scales, sb, pad=pad[2])
    c = Window(hb, out, c0, pad=pad[2], offset=offset)
    hb.gemm_blocks(a.t, wsa.t, B.transpose_matrix(b.t), wsb.t, c.t, alpha, beta)
    with np.errstate(invalid="ignore"):
        va, vb = H.unquantized(qa, sa, ba, scales), H.unquantized(qb, sb, bb, scales)
        want = alpha * (va @ vb.T)
        size = abs(alpha) * (np.abs(va) @ np.abs(vb).T)
        if beta:
            want, size = want + beta * H.values(c0, out), size + abs(beta) * np.abs(H.values(c0, out))
    size = np.where(np.isfinite(size), size, 0.0)
    blocks = -(-k // 128)
    close(H.values(c.read(), out), want, (128 + 2 * blocks + 3) * 2.0 ** -24 * size + H.SMALL[out] * H.ROUNDING[out], 1.01 * H.ROUNDING[out], "c")


@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("ba,bb", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 128), (2, 17, 300), (17, 129, 127), (33, 256, 256), (65, 300, 1000), (200, 513, 384), (130, 1, 640)])
def test_gemm_blocks(hb, m, n, k, ba, bb, scales):
    out = [F32, BF16, F16][(m + n + k) % 3]
    product(hb, rng(200 + m), m, n, k, scales, ba, bb, out)


@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("pad,offset", [((0, 0, 0), 0), ((16, 32, 4), 0), ((1, 3, 1), 1), ((16, 16, 16), 16), ((8, 8, 2), 8)])
@pytest.mark.parametrize("m", [1, 5, 40, 150, 300])
def test_gemm_blocks_pitches_and_offsets(hb, m, pad, offset, scales):
    for out in (F32, BF16, F16):
        product(hb, rng(300 + m), m, 264, 272, scales, 1, 128, out, pad=pad, offset=offset)


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("m", [1, 70, 260])
def test_gemm_blocks_alpha_and_beta(hb, m, out):
    for alpha, beta in ((0.5, 0.0), (1.0, 1.0), (-2.0, 0.25), (0.0, 3.0), (0.0, 0.0)):
        product(hb, rng(400 + m), m, 260, 256, F32, 1, 128, out, alpha, beta)


@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (8, 2048, 8192), (31, 1024, 2048), (64, 512, 1024), (512, 512, 4096), (512, 768, 512), (1000, 1500, 400)])
def test_gemm_blocks_larger(hb, m, n, k, scales):
    product(hb, rng(500 + m), m, n, k, scales, 1, 128, F32)
    product(hb, rng(501 + m), m, n, k, scales, 1, 1, BF16)


@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("m", [3, 200, 512])
def test_gemm_blocks_carries_what_is_not_a_number(hb, m, scales):
    """A block with an infinity or NaN spoils the outputs that read it, and no other."""
    def spoil(a, b):
        a[1, 130] = np.inf
        b[7, 5] = np.nan
    product(hb, rng(600), m, 256, 256, scales, 1, 1, F32, spoil=spoil)


PLANS = [
    # m, n, k, out, the kernel that the plan's cost picks
    (9, 600, 128, F32, "thin"), (5, 70, 100, BF16, "thin"), (40, 1024, 1024, F32, "bf16_16x16"), (3, 1000, 700, F32, "bf16_16x16_any"),
    (33, 1000, 301, F32, "bf16_16x16_any"), (60, 2201, 1040, F32, "bf16_32x32"), (3, 5000, 530, F32, "bf16_32x32_any"),
    (257, 1000, 1040, F32, "bf16_32x64"), (2074, 17, 257, BF16, "bf16_32x64_any"), (90, 3000, 530, F32, "bf16_32x64_any"),
    (16, 8200, 256, BF16, "thin"), (1024, 1024, 256, F32, "bf16_64x64"), (300, 900, 200, F32, "bf16_64x64_any"),
    (2048, 2560, 272, F32, "bf16_128x128"), (1030, 1001, 127, F32, "bf16_128x128_any"), (2049, 2561, 201, F16, "bf16_128x128_any"),
    (60, 2201, 1040, F16, "fp8_32x32"), (40, 1501, 1041, F16, "fp8_32x32_any"), (130, 2100, 1040, BF16, "fp8_32x64"),
    (65, 4099, 1300, F16, "fp8_32x64_any"), (1024, 2048, 528, BF16, "fp8_64x64"), (500, 1030, 530, BF16, "fp8_64x64_any"),
    (2048, 2048, 560, F16, "fp8_128x128"), (2050, 4099, 515, BF16, "fp8_128x128_any"), (4100, 4090, 528, BF16, "fp8_256x256"),
    (4090, 4082, 528, BF16, "fp8_256x256"),
]


@pytest.mark.parametrize("scales,ba,bb", [(F32, 1, 128), (F32, 128, 1), (E8M0, 1, 1)])
@pytest.mark.parametrize("m,n,k,out,kernel", PLANS)
def test_gemm_blocks_on_every_kernel(hb, m, n, k, out, kernel, scales, ba, bb):
    product(hb, rng(700 + m), m, n, k, scales, ba, bb, out)
    assert hb.debug_launches()[-1] == "gemm_blocks_" + kernel


@pytest.mark.parametrize("m,n,k,out,kernel", PLANS)
def test_gemm_blocks_on_every_kernel_into_what_is_there(hb, m, n, k, out, kernel):
    """beta, and rows of C at an odd pitch and offset."""
    any_address = kernel.endswith("_any")
    product(hb, rng(710 + m), m, n, k, F32, 1, 128, out, 0.5, -1.0, pad=(1, 2, 3) if any_address else (0, 16, 3))


@pytest.mark.parametrize("scales", [F32, E8M0])
@pytest.mark.parametrize("m,n,k", [(200, 256, 640), (2050, 300, 515), (5, 200, 700)])
def test_gemm_blocks_carries_what_is_not_a_number_into_16_bits(hb, m, n, k, scales):
    def spoil(a, b):
        a[1, 130] = np.inf
        b[7, 5] = np.nan
    product(hb, rng(630 + m), m, n, k, scales, 1, 1, BF16, spoil=spoil)


@pytest.mark.parametrize("m,n,k", [(3, 200, 256), (200, 256, 256), (40, 70, 131)])
def test_gemm_blocks_of_any_scale(hb, m, n, k):
    """Rows whose sizes differ by 150 powers of two; products of two scales stay normal f32 numbers."""
    g = rng(640 + m)
    for scales in (F32, E8M0):
        def spoil(a, b):
            a *= np.exp2(g.integers(-60, 90, (m, 1))).astype(np.float32)
            b *= np.float32(2.0 ** -30)
        product(hb, g, m, n, k, scales, 1, 1, F32, spoil=spoil)


def test_gemm_blocks_without_a_sum(hb):
    """K = 0 and alpha = 0: c = beta * c; alpha = 0 reads neither operand (here full of NaN)."""
    g = rng(610)
    c0 = g.standard_normal((5, 9)).astype(np.float32)
    for beta in (0.0, 2.0):
        c = Window(hb, F32, c0)
        a, b = Window(hb, E4M3, shape=(5, 0)), Window(hb, E4M3, shape=(9, 0))
        sa, sb = Window(hb, F32, shape=(5, 0)), Window(hb, F32, shape=(9, 0))
        hb.gemm_blocks(a.t, sa.t, B.transpose_matrix(b.t), sb.t, c.t, 1.0, beta)
        assert np.array_equal(c.read(), np.float32(beta) * c0)
    nan = np.full((5, 128), 127, np.uint8)
    a, b, c = Window(hb, E4M3, nan), Window(hb, E4M3, np.full((9, 128), 127, np.uint8)), Window(hb, F32, c0)
    sa, sb = Window(hb, F32, np.ones((5, 1), np.float32)), Window(hb, F32, np.ones((9, 1), np.float32))
    hb.gemm_blocks(a.t, sa.t, B.transpose_matrix(b.t), sb.t, c.t, 0.0, 2.0)
    assert np.array_equal(c.read(), np.float32(2.0) * c0)


def test_gemm_blocks_repeats_its_bits(hb):
    """The same product twice, with other work between, gives the same bits."""
    g = rng(620)
    qa, sa = H.quantize(g.standard_normal((24, 4096)).astype(np.float32), 1, F32)
    qb, sb = H.quantize(g.standard_normal((300, 4096)).astype(np.float32), 128, F32)
    ops = [Window(hb, E4M3, qa), Window(hb, F32, sa), Window(hb, E4M3, qb), Window(hb, F32, sb)]
    got = []
    for _ in range(3):
        c = Window(hb, F32, shape=(24, 300))
        hb.gemm_blocks(ops[0].t, ops[1].t, B.transpose_matrix(ops[2].t), ops[3].t, c.t)
        got.append(c.read().view(np.uint32))
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


# ------------------------------------------------------------------------------ log probs


LOWEST = {F32: -3.4028235e38, F16: -65504.0, BF16: -3.3895314e38}


def logits(g, r, v, dtype, masks=True):
    """Rows as they come: loud ones, masked ones, an empty one, one of the type's lowest value."""
    x = 3.0 * g.standard_normal((r, v)) + 2.0 * np.exp(g.standard_normal((r, v)) - 1.0)
    if masks and v > 1:
        x[:, v - max(1, v // 50):] = -np.inf
        if r > 1:
            x[1, ::2] = LOWEST[dtype]
        if r > 2:
            x[2] = -np.inf
        if r > 3:
            x[3] = LOWEST[dtype]
        if r > 4:
            x[4], x[4, v // 2] = -np.inf, 1.25
    return H.to_bits(x, dtype)


def check_logprobs(hb, bits, dtype, tokens, k, t, pad=0, offset=0):
    r, v = bits.shape
    x = Window(hb, dtype, bits, pad=pad, offset=offset)
    tok = Window(hb, I32, tokens)
    lp, h, st = Window(hb, F32, shape=[r]), Window(hb, F32, shape=[r]), Window(hb, F32, shape=[r, 2], pad=1)
    top = Window(hb, F32, shape=[r, k], pad=2) if k else None
    ids = Window(hb, I32, shape=[r, k], pad=1, offset=1) if k else None
    hb.token_logprobs(x.t, tok.t, t, lp.t, h.t, st.t, top.t if k else None, ids.t if k else None)
    num = H.values(bits, dtype)
    want = H.logprobs(num, tokens, k, t)
    eps = 2.0 ** -23
    close(lp.read(), want[0], TOL, 4 * eps, "logprobs")
    close(h.read(), want[1], TOL_ENTROPY, 4 * eps, "entropy")
    got = st.read()
    close(got[:, 0], want[2][:, 0], 0.0, 0.0, "largest")
    close(got[:, 1], want[2][:, 1], TOL, eps, "log sum")
    if k:
        assert np.array_equal(ids.read(), want[4])
        close(top.read(), want[3], TOL, 4 * eps, "top")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r,v", [(1, 1), (2, 2), (5, 7), (6, 8), (7, 9), (3, 1000), (9, 4097), (5, 50001), (2, 140001), (1, 300007), (600, 333), (530, 5000)])
def test_token_logprobs(hb, r, v, dtype):
    g = rng(700 + v)
    tokens = g.integers(0, v, r).astype(np.int32)
    tokens[1::7] = -1
    tokens[3::7] = v
    check_logprobs(hb, logits(g, r, v, dtype), dtype, tokens, [1, 5, 20, 128][(r + v) % 4], [1.0, 0.5, 3.0][v % 3])


@pytest.mark.parametrize("k", [0, 1, 2, 64, 127, 128])
@pytest.mark.parametrize("v", [3, 100, 1025, 70000])
def test_token_logprobs_alternatives(hb, v, k):
    g = rng(800 + v)
    check_logprobs(hb, logits(g, 4, v, BF16), BF16, g.integers(0, v, 4).astype(np.int32), k, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (3, 2), (5, 7), (8, 8)])
def test_token_logprobs_pitches_and_offsets(hb, pad, offset, dtype):
    g = rng(900 + pad)
    for r, v in ((3, 801), (520, 130)):
        check_logprobs(hb, logits(g, r, v, dtype), dtype, g.integers(0, v, r).astype(np.int32), 9, 1.0, pad, offset)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r,v", [(1, 40000), (2, 9000), (513, 9000)])
def test_token_logprobs_of_equal_logits(hb, r, v, dtype):
    """Ties go to the lowest index: constant rows, rows of two values, rising and falling rows, zeros of both signs."""
    x = np.zeros((r, v))
    for i in range(r):
        x[i] = [np.full(v, 1.5), (np.arange(v) % 3 == 1) * 2.0, np.floor(np.arange(v) / 700.0), -np.floor(np.arange(v) / 700.0),
                np.where(np.arange(v) % 2 == 0, -0.0, 0.0), np.where(np.arange(v) < v - 40, -np.inf, -3.0)][(i + v) % 6]
    tokens = np.full(r, v - 1, np.int32)
    for k in (1, 20, 128):
        check_logprobs(hb, H.to_bits(x, dtype), dtype, tokens, k, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v,k", [(600, 128), (1000, 128), (1999, 128), (500, 24), (16000, 128)])
@pytest.mark.parametrize("r", [3, 130, 1100])
def test_token_logprobs_of_rows_that_stay_candidates(hb, r, v, k, dtype):
    """Fewer slots than alternatives, or most elements equal: nearly all of a row's elements are looked at."""
    g = rng(950 + v)
    x = g.standard_normal((r, v)) * 3
    x[::3] = g.integers(0, 2, x[::3].shape)
    x[1::3, v // 3:] = -5.0
    check_logprobs(hb, H.to_bits(x, dtype), dtype, g.integers(0, v, r).astype(np.int32), k, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r,v", [(2, 9000), (3, 70000), (1100, 4000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_token_logprobs_of_logits_a_unit_apart(hb, sign, r, v, dtype):
    """Eight neighbouring numbers of the type, so that what tells the alternatives is the last bits and the ids."""
    g = rng(970 + v)
    x = sign * (1.0 + g.integers(0, 8, (r, v)) * 2.0 ** {F32: -23, F16: -10, BF16: -7}[dtype])
    for k in (5, 24, 128):
        check_logprobs(hb, H.to_bits(x, dtype), dtype, g.integers(0, v, r).astype(np.int32), k, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_token_logprobs_of_a_peak(hb, dtype):
    """Almost all of the probability on one logit: the small entropy keeps its digits."""
    g = rng(1000)
    x = g.standard_normal((4, 30000))
    x[np.arange(4), [0, 17, 29999, 15000]] = [14.0, 22.0, 30.0, 60.0]
    bits = H.to_bits(x, dtype)
    w, h = Window(hb, dtype, bits), Window(hb, F32, shape=[4])
    hb.token_logprobs(w.t, entropy=h.t)
    want = H.logprobs(H.values(bits, dtype), np.full(4, -1), 0, 1.0)[1]
    # The peak's own eight are summed in f32: 4 * 2^-24 and the rounding of the result; the others' sums lose 1e-5 of themselves.
    close(h.read(), want, 2.0 ** -22, 2e-5, "entropy")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r,v", [(4, 77), (3, 30000), (515, 300)])
def test_token_logprobs_of_what_is_not_a_number(hb, r, v, dtype):
    g = rng(1100)
    num = np.array(H.values(logits(g, r, v, dtype, masks=False), dtype))
    num[0, v // 2], num[1, v - 1], num[2, 0] = np.nan, np.inf, -np.nan
    num[2, 1:] = -np.inf
    bits = H.to_bits(num, dtype)
    tokens = np.arange(r, dtype=np.int32) % 3 - 1
    check_logprobs(hb, bits, dtype, tokens, 7, 1.0)


def test_token_logprobs_of_nothing(hb):
    """No rows, and rows without logits."""
    x = Window(hb, F32, shape=[0, 50])
    lp, tok = Window(hb, F32, shape=[0]), Window(hb, I32, shape=[0])
    hb.token_logprobs(x.t, tok.t, 1.0, lp.t)
    x, h, st = Window(hb, F32, shape=[3, 0]), Window(hb, F32, shape=[3]), Window(hb, F32, shape=[3, 2])
    top, ids = Window(hb, F32, shape=[3, 2]), Window(hb, I32, shape=[3, 2])
    hb.token_logprobs(x.t, None, 1.0, None, h.t, st.t, top.t, ids.t)
    assert not h.read().any() and np.all(st.read() == -np.inf) and np.all(ids.read() == -1) and np.all(top.read() == -np.inf)


def bound(coefficient, want, dtype):
    """atol of a gradient: 1e-5 of the row's coefficient, and half a unit of the type around zero."""
    return 1e-5 * np.abs(coefficient)[:, None] + H.SMALL[dtype] * H.ROUNDING[dtype] + 0 * np.where(np.isfinite(want), want, 0)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r,v,pad,offset", [(1, 1, 0, 0), (5, 9, 1, 3), (6, 1000, 0, 0), (7, 8193, 3, 1), (2, 40001, 0, 0)])
def test_token_logprobs_backward(hb, r, v, pad, offset, dtype, inplace):
    g = rng(1200 + v)
    bits = logits(g, r, v, dtype)
    tokens = g.integers(0, v, r).astype(np.int32)
    tokens[2::5] = -1
    t = [1.0, 0.5, 2.0][v % 3]
    num = H.values(bits, dtype)
    x = Window(hb, dtype, bits, pad=pad, offset=offset)
    tok, h, st = Window(hb, I32, tokens), Window(hb, F32, shape=[r]), Window(hb, F32, shape=[r, 2])
    hb.token_logprobs(x.t, None, t, None, h.t, st.t)
    glp, gh = g.standard_normal(r).astype(np.float32), g.standard_normal(r).astype(np.float32)
    wg, wh = Window(hb, F32, glp), Window(hb, F32, gh)
    for with_entropy in ((True,) if inplace else (False, True)):
        dx = x if inplace else Window(hb, dtype, shape=[r, v], pad=pad, offset=offset + 1)
        hb.token_logprobs_backward(x.t, tok.t, t, st.t, h.t if with_entropy else None, wg.t, wh.t if with_entropy else None, dx.t)
        want = H.logprobs_backward(num, tokens, t, glp.astype(float), gh.astype(float) * with_entropy)
        size = (np.abs(glp) + np.abs(gh) * with_entropy * (np.log(v) + 5)) / t
        close(H.values(dx.read(), dtype), want, bound(size, want, dtype), 1.01 * H.ROUNDING[dtype], "dlogits")


def test_token_logprobs_backward_of_what_is_not_a_number(hb):
    x0 = np.array([[1.0, np.nan, 2.0], [np.inf, 0.0, 0.0], [-np.inf] * 3, [0.0, -np.inf, 1.0]], np.float32)
    x, tok = Window(hb, F32, x0), Window(hb, I32, np.array([0, -1, 1, 0], np.int32))
    h, st, dx = Window(hb, F32, shape=[4]), Window(hb, F32, shape=[4, 2]), Window(hb, F32, shape=[4, 3])
    one = Window(hb, F32, np.ones(4, np.float32))
    hb.token_logprobs(x.t, None, 1.0, None, h.t, st.t)
    hb.token_logprobs_backward(x.t, tok.t, 1.0, st.t, h.t, one.t, one.t, dx.t)
    got = dx.read()
    assert np.isnan(got[:2]).all() and not got[2].any()
    close(got[3:], H.logprobs_backward(x0[3:].astype(float), [0], 1.0, [1.0], [1.0]), 1e-6, 1e-6, "the fine row")


def differences(f, x, at, eps=1e-5):
    """Central differences of a 64-bit function in the places `at`."""
    out = []
    for i in at:
        up, down = x.copy(), x.copy()
        up[i] += eps
        down[i] -= eps
        out.append((f(up) - f(down)) / (2 * eps))
    return np.array(out)


def test_gradients_against_differences(hb):
    """Both gradients against central differences of the 64-bit losses (their error: about 1e-9)."""
    g = rng(1300)
    r, v, t, k = 3, 200, 1.5, 12
    x0 = (2.0 * g.standard_normal((r, v))).astype(np.float32)
    tokens = np.array([5, 199, 0], np.int32)
    glp, gh = np.array([1.0, -0.5, 2.0], np.float32), np.array([0.3, 0.0, -1.0], np.float32)
    ids = np.stack([g.permutation(v)[:k] for _ in range(r)]).astype(np.int32)
    lists = np.log(g.dirichlet(np.ones(k + 5), r)[:, :k]).astype(np.float32)
    weights = np.array([1.0, 0.25, 3.0], np.float32)
    x, tok, h, st = Window(hb, F32, x0), Window(hb, I32, tokens), Window(hb, F32, shape=[r]), Window(hb, F32, shape=[r, 2])
    wg, wh, dx = Window(hb, F32, glp), Window(hb, F32, gh), Window(hb, F32, shape=[r, v])
    hb.token_logprobs(x.t, None, t, None, h.t, st.t)
    hb.token_logprobs_backward(x.t, tok.t, t, st.t, h.t, wg.t, wh.t, dx.t)
    places = [(i, j) for i in range(r) for j in [*ids[i][:4], tokens[i], 17, 100]]

    def policy(y):
        lp, ent, *_ = H.logprobs(y, tokens, 0, t)
        return (glp * lp).sum() + (gh * ent).sum()
    got = dx.read()
    close([got[p] for p in places], differences(policy, x0.astype(float), places), 2e-5, 1e-5, "dlogits")
    for normalize in (False, True):
        losses, dl = Window(hb, F32, shape=[r]), Window(hb, F32, shape=[r, v])
        hb.distill_grad(x.t, Window(hb, I32, ids).t, Window(hb, F32, lists).t, Window(hb, F32, weights).t, t, normalize, losses.t, dl.t)
        want = differences(lambda y: H.distill(y, ids, lists, weights, t, normalize)[0].sum(), x0.astype(float), places)
        got = dl.read()
        close([got[p] for p in places], want, 5e-5, 1e-5, "dlogits")


# --------------------------------------------------------------------------------- distill


def teacher(g, r, v, k):
    ids = np.stack([g.permutation(v)[:k] if v >= k else np.resize(g.permutation(v), k) for _ in range(r)]).astype(np.int32)
    if v < k:
        ids[:, v:] = -1
    lists = np.log(g.dirichlet(np.full(k + 3, 0.3), r)[:, :k] + 1e-30).astype(np.float32)
    if k > 2:
        ids[0, k // 2] = -1
        lists[0, k // 2] = np.nan  # behind an id that names nothing: not looked at
        lists[-1, 0] = -np.inf
        ids[-1, 1] = v
    return ids, lists


def check_distill(hb, bits, dtype, ids, lists, weights, t, normalize, pad=0, offset=0, inplace=False, grad=True):
    r, v = bits.shape
    x = Window(hb, dtype, bits, pad=pad, offset=offset)
    wi, wl = Window(hb, I32, ids, pad=1), Window(hb, F32, lists, pad=3)
    ww = Window(hb, F32, weights) if weights is not None else None
    losses = Window(hb, F32, shape=[r])
    dx = None if not grad else x if inplace else Window(hb, dtype, shape=[r, v], pad=pad + 1, offset=offset)
    hb.distill_grad(x.t, wi.t, wl.t, ww.t if ww else None, t, normalize, losses.t, dx.t if grad else None)
    w = np.ones(r) if weights is None else weights.astype(float)
    num = H.values(bits, dtype)
    want_loss, want = H.distill(num, ids, lists, w, t, normalize)
    with np.errstate(over="ignore"):
        want_loss = want_loss.astype(np.float32)  # a lowest-value mask that the teacher likes can cost more than f32 holds
    lp_size = np.where(np.isfinite(num), np.abs(num), 0).max(1, initial=0).clip(0, 1e4) / t + np.log(v + 1) + 10
    mass = 1.0 if normalize else np.exp(np.where(np.isfinite(lists) & (ids >= 0), lists, -np.inf).astype(float)).sum(1).clip(1)
    close(losses.read(), want_loss, np.abs(w) * t * t * mass * (TOL + 2.0 ** -22 * lp_size), 1e-6, "losses")
    if grad:
        # The teacher's own p is off by 2^-23 of |log p| at most: 1e-5 for what matters of it.
        close(H.values(dx.read(), dtype), want, bound(2 * w * t * mass, want, dtype), 1.01 * H.ROUNDING[dtype], "dlogits")


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r,v,k", [(1, 1, 1), (5, 9, 4), (6, 8, 12), (3, 1000, 64), (7, 8195, 128), (2, 70001, 20), (1, 300007, 5), (600, 333, 9), (530, 5003, 33)])
def test_distill_grad(hb, r, v, k, dtype, normalize):
    g = rng(1400 + v)
    ids, lists = teacher(g, r, v, k)
    weights = g.uniform(0.1, 2.0, r).astype(np.float32)
    weights[3::4] = 0.0
    check_distill(hb, logits(g, r, v, dtype), dtype, ids, lists, weights, [1.0, 0.5, 2.0][v % 3], normalize)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 2), (7, 5), (8, 8)])
def test_distill_grad_pitches_and_in_place(hb, pad, offset, dtype):
    g = rng(1500 + pad)
    for r, v in ((3, 2001), (515, 200), (520, 9001)):
        ids, lists = teacher(g, r, v, 17)
        bits = logits(g, r, v, dtype)
        for inplace in (False, True):
            check_distill(hb, bits, dtype, ids, lists, None, 2.0, True, pad, offset, inplace)


@pytest.mark.parametrize("r", [4, 520])
def test_distill_grad_edges(hb, r):
    """Losses alone; an id given twice; a list of nothing; no list at all."""
    g = rng(1600)
    v = 500
    bits = logits(g, r, v, BF16)
    ids, lists = teacher(g, r, v, 6)
    check_distill(hb, bits, BF16, ids, lists, None, 1.0, True, grad=False)
    ids[:, 5] = ids[:, 3]
    ids[0] = -1
    check_distill(hb, bits, BF16, ids, lists, None, 1.0, False)
    check_distill(hb, bits, BF16, ids, lists, None, 1.0, True)
    x, losses, dx = Window(hb, BF16, bits), Window(hb, F32, shape=[r]), Window(hb, BF16, shape=[r, v])
    none, empty = Window(hb, I32, shape=[r, 0]), Window(hb, F32, shape=[r, 0])
    hb.distill_grad(x.t, none.t, empty.t, None, 1.0, True, losses.t, dx.t)
    assert not losses.read().any() and not H.values(dx.read(), BF16).any()


@pytest.mark.parametrize("r", [6, 520])
def test_distill_grad_of_what_is_not_a_number(hb, r):
    """NaN and +inf spoil their row, unless it has no weight or no list; a masked logit that the teacher likes costs +inf."""
    g = rng(1700)
    v = 300
    x = np.array(H.values(logits(g, r, v, F32, masks=False), F32))
    x[0, 9], x[1, 250], x[2, 3], x[3, 7] = np.nan, np.inf, np.nan, np.nan
    ids, lists = teacher(g, r, v, 5)
    ids[3] = -1
    x[5, ids[5, 2]] = -np.inf
    weights = np.ones(r, np.float32)
    weights[2] = 0.0
    check_distill(hb, H.to_bits(x, F32), F32, ids, lists, weights, 1.0, True)


# -------------------------------------------------------------------- streams and capture


def test_rows_split_over_workgroups_on_two_streams(hb):
    """Calls that share the context's scratch, on two streams in turn, as one stream would give them."""
    import ctypes

    from linalg_hip import _native as N
    g = rng(1800)
    bits = logits(g, 2, 100000, BF16, masks=False)
    x = Window(hb, BF16, bits)
    q = hb.ctx.new_stream()
    want = H.logprobs(H.values(bits, BF16), [0, 0], 20, 1.0)
    outs = [(Window(hb, F32, shape=[2, 20]), Window(hb, I32, shape=[2, 20])) for _ in range(8)]
    hb.sync()
    for i, (top, ids) in enumerate(outs):
        refs = [ctypes.byref(w.t.to_c()) for w in (top, ids)]
        assert N.lib().lg_backend_token_logprobs(hb.ctx.handle, q.handle if i % 2 else None, ctypes.byref(x.t.to_c()), None, 1.0, None, None,
                                                 None, *refs) == 0
    q.wait_until_completed()
    for top, ids in outs:
        assert np.array_equal(ids.read(), want[4])
        close(top.read(), want[3], TOL, 1e-6, "top")
    q.close()
