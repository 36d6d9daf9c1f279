// gfx950 kernels of gemm_blocks: C = alpha * sum over blocks b of sa[m, b] sb[n, b] (A_b . B_b^T) + beta * C
// of e4m3 operands with a scale for each 128 columns of K and each row, or each 128 rows.
//
// The fp8 matrix instructions align each eight neighbouring products to the largest of them and keep 2^-13 of
// it (measured: 1.5e-5 of the norm for normal operands, 1.2e-5 of the sum of absolute products at K = 128).
// gemm_blocks_any therefore turns elements into bf16, which holds every e4m3 value, two to an instruction on
// their way from LDS, and multiplies on v_mfma_f32_16x16x32_bf16: four of those are a block's sum for 16x16
// outputs, exact products summed in f32 (7e-8 of the norm at K = 4096). The instructions' order of K is free
// as long as both operands share it: a lane takes 32 bytes of one row of each operand (row lane % 16, the
// quarter of the block goes by lane / 16) and eight of them per instruction. B's rows are the first operand and
// A's the second, so a lane's four outputs are neighbours along N of one row of C. A block's sums start
// at zero and join the f32 accumulator by a multiply-add with sa * sb.
#include "head_device.h"

namespace lg {
namespace {

using namespace head_detail;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int THREADS = 256;

// Eight e4m3 elements as bf16, which holds each of them.
__device__ inline bf16x8 to_bf16(uint32_t lo, uint32_t hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's part of a row in a block of 128: 32 elements.
struct Fragment {
    bf16x8 v[4];
    __device__ inline Fragment() {}
    __device__ inline Fragment(u32x4 lo, u32x4 hi) : v{to_bf16(lo[0], lo[1]), to_bf16(lo[2], lo[3]), to_bf16(hi[0], hi[1]), to_bf16(hi[2], hi[3])} {}
};

// A block's sums for 16x16 outputs.
__device__ inline f32x4 block_product(const Fragment& b, const Fragment& a) {
    f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[i], a.v[i], p, 0, 0, 0);
    return p;
}

__device__ inline float e8m0_value(uint32_t code) {
    // 2^-127, code 0, is subnormal.
    return code == 255 ? __builtin_nanf("") : __uint_as_float(code == 0 ? 0x400000u : code << 23);
}

// The scale of row `row` in block `kb`.
template <bool E8M0, int BLOCK>
__device__ inline float scale_at(const void* s, int64_t pitch, uint32_t row, uint32_t kb) {
    const int64_t at = static_cast<int64_t>(BLOCK == 1 ? row : row / BLOCK_K) * pitch + kb;
    if constexpr (E8M0) {
        return e8m0_value(static_cast<const uint8_t*>(s)[at]);
    } else {
        return static_cast<const float*>(s)[at];
    }
}

// Bytes k .. k + 15 of a row of length K at any address, zeros past its end.
__device__ inline u32x4 load_sixteen(const uint8_t* row, uint32_t k, uint32_t K) {
    if (k + 16 <= K) return *reinterpret_cast<const u32x4_any*>(row + k);
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (k + i < K) v[i / 4] |= static_cast<uint32_t>(row[k + i]) << (8 * (i % 4));
    }
    return v;
}

// Outputs (m, n .. n + 3), those inside C, from the sums of a lane.
template <uint32_t OUT>
__device__ inline void store_four(const GemmBlocksArgs& g, uint32_t m, uint32_t n, f32x4 acc) {
    if (m >= g.m || n >= g.n) return;
    char* p = static_cast<char*>(g.c) + (m * g.c_pitch + n) * elem_size<OUT>;
    float v[4];
    const uint32_t inside = min(g.n - n, 4u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = g.alpha * acc[e];
        if (g.beta != 0.0f && static_cast<uint32_t>(e) < inside) v[e] = v[e] + g.beta * load_one<OUT>(p + e * elem_size<OUT>);
    }
    if (inside == 4) {
        if constexpr (OUT == LG_DTYPE_F32) {
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __float_as_uint(v[e]);
            *reinterpret_cast<u32x4_any*>(p) = o;
        } else {
            *reinterpret_cast<u32x2_any*>(p) = u32x2{pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3])};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (static_cast<uint32_t>(e) < inside) store_one<OUT>(p + e * elem_size<OUT>, v[e]);
        }
    }
}

// A 128x128 tile of C by four waves of 64x64, operands at any address: slices of 128 columns pass
// through registers into LDS, [row][128] with 16-byte chunk c of row r at place c ^ (r & 7), so that
// eight neighbouring rows' reads of one chunk touch every bank once.
constexpr int TILE = 128;

template <uint32_t OUT, bool E8M0, int BA, int BB>
__global__ __launch_bounds__(THREADS) void gemm_blocks_any(GemmBlocksArgs g, uint32_t tiles_m) {
    __shared__ u32x4 lds[2][TILE * 8];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const uint32_t m0 = (blockIdx.x % tiles_m) * TILE, n0 = (blockIdx.x / tiles_m) * TILE;
    const uint32_t wm = (wave % 2) * 64, wn = (wave / 2) * 64;
    const uint32_t chunk = tid % 8, line = tid / 8, blocks = (g.k + BLOCK_K - 1) / BLOCK_K;
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    u32x4 ra[4], rb[4];
    // Rows past the operand's last one repeat it: their outputs are not stored.
    auto fetch = [&](uint32_t kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = line + 32 * i;
            ra[i] = load_sixteen(g.a + min(m0 + r, g.m - 1) * g.a_pitch, kb * BLOCK_K + chunk * 16, g.k);
            rb[i] = load_sixteen(g.b + min(n0 + r, g.n - 1) * g.b_pitch, kb * BLOCK_K + chunk * 16, g.k);
        }
    };
    auto fragment = [&](int op, uint32_t r) {
        const u32x4 lo = lds[op][r * 8 + ((lane / 16) ^ (r & 7))], hi = lds[op][r * 8 + ((lane / 16 + 4) ^ (r & 7))];
        return Fragment(lo, hi);
    };
    if (blocks > 0) fetch(0);
    for (uint32_t kb = 0; kb < blocks; ++kb) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = line + 32 * i;
            lds[0][r * 8 + (chunk ^ (r & 7))] = ra[i];
            lds[1][r * 8 + (chunk ^ (r & 7))] = rb[i];
        }
        __syncthreads();
        if (kb + 1 < blocks) fetch(kb + 1);
        Fragment fa[4];
        float sa[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            fa[j] = fragment(0, wm + 16 * j + lane % 16);
            sa[j] = scale_at<E8M0, BA>(g.sa, g.sa_pitch, min(m0 + wm + 16 * j + lane % 16, g.m - 1), kb);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Fragment fb = fragment(1, wn + 16 * i + lane % 16);
            float sb[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sb[e] = scale_at<E8M0, BB>(g.sb, g.sb_pitch, min(n0 + wn + 16 * i + (lane / 16) * 4 + e, g.n - 1), kb);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 p = block_product(fb, fa[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(sa[j] * sb[e], p[e], acc[i][j][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            store_four<OUT>(g, m0 + wm + 16 * j + lane % 16, n0 + wn + 16 * i + (lane / 16) * 4, acc[i][j]);
        }
    }
}

// The same product of operands that allow 16-byte copies (bases, pitches and K in whole 16 bytes): a
// TM x TN tile of C by WM x WN waves, slices of 128 columns copied from memory straight into LDS
// (global_load_lds_dwordx4, [row][128] with the places of gemm_blocks_any) while the slice before is
// multiplied. A slice's scales pass through registers into LDS beside it, one a thread.
// FAST multiplies on v_mfma_f32_16x16x128_f8f6f4, one instruction to a block of 16x16 outputs, at the
// precision above; e8m0 scales are then the instruction's own operands.
__device__ inline void copy_sixteen(const uint8_t* src, uint8_t* lds) { __builtin_amdgcn_global_load_lds(src, lds, 16, 0, 0); }

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <bool FAST>
struct Operand {
    typedef Fragment T;
};
template <>
struct Operand<true> {
    struct T {
        i32x8 v;
        __device__ inline T() {}
        __device__ inline T(u32x4 lo, u32x4 hi) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = static_cast<int>(lo[i]);
                v[i + 4] = static_cast<int>(hi[i]);
            }
        }
    };
};

// Workgroup `id` of `count` to a tile: neighbouring ids go to the eight XCDs in turn, so each XCD takes one
// run of tiles, and runs walk bands of eight tiles along M, whose operands its L2 then holds.
__device__ inline void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t* tm, uint32_t* tn) {
    constexpr uint32_t XCDS = 8, BAND = 8;
    const uint32_t count = tiles_m * tiles_n, per = count / XCDS, left = count % XCDS, xcd = id % XCDS;
    const uint32_t t = xcd * per + min(xcd, left) + id / XCDS;
    const uint32_t band = t / (BAND * tiles_n), first = band * BAND, high = min(BAND, tiles_m - first), in = t - first * tiles_n;
    *tm = first + in % high;
    *tn = in / high;
}

template <uint32_t OUT, bool FAST, bool E8M0, bool BROWS, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void gemm_blocks_tile(GemmBlocksArgs g, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int WAVES = WM * WN, T = WAVES * 64, FM = TM / WM / 16, FN = TN / WN / 16;
    constexpr int STAGE = (TM + TN) * 128, COPIES = STAGE / 16 / T;  // copies a thread; A's rows first
    constexpr bool HARDWARE = FAST && E8M0;
    static_assert(BROWS || (TN / WN) % 128 == 0 || 128 % (TN / WN) == 0, "a wave's columns share their scale");
    __shared__ __attribute__((aligned(16))) uint8_t stages[2][STAGE];
    __shared__ __attribute__((aligned(16))) float scales[2][TM + TN];  // or e8m0 codes
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    uint32_t tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
    const uint32_t m0 = tm * TM, n0 = tn * TN, wm = (wave % WM) * (TM / WM), wn = (wave / WM) * (TN / WN);
    const uint32_t blocks = (g.k + BLOCK_K - 1) / BLOCK_K;
    const uint8_t* pa = g.a + static_cast<int64_t>(m0) * g.a_pitch;
    const uint8_t* pb = g.b + static_cast<int64_t>(n0) * g.b_pitch;
    // Copy i of a wave: 1 KB of a stage, eight rows. Rows past the operand's last one repeat it.
    static_assert(TM % (WAVES * 8) == 0 && TN % (WAVES * 8) == 0, "a copy is of one operand");
    uint32_t offset[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const uint32_t r = (i * WAVES + wave) * 8 + lane / 8, chunk = (lane % 8) ^ (r & 7);
        const bool of_a = i * WAVES * 8 < TM;
        const uint32_t row = of_a ? min(r, g.m - 1 - m0) : min(r - TM, g.n - 1 - n0);
        offset[i] = row * static_cast<uint32_t>(of_a ? g.a_pitch : g.b_pitch) + chunk * 16;
    }
    auto copy = [&](uint32_t kb) {
        const uint32_t left = g.k - kb * BLOCK_K;
        uint8_t* stage = stages[kb % 2] + wave * 1024;
        const uint8_t* a = pa + kb * BLOCK_K;
        const uint8_t* b = pb + kb * BLOCK_K;
        if (left >= BLOCK_K) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) copy_sixteen((i * WAVES * 8 < TM ? a : b) + offset[i], stage + i * WAVES * 1024);
        } else {
            const uint32_t lane_chunk = ((lane % 8) ^ (lane / 8)) * 16;  // of every copy: eight rows at a time
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                if (lane_chunk < left) {
                    copy_sixteen((i * WAVES * 8 < TM ? a : b) + offset[i], stage + i * WAVES * 1024);
                } else {
                    *reinterpret_cast<u32x4*>(stage + i * WAVES * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
                }
            }
        }
    };
    // Thread t holds the scale of row t of the tile's operands (A's rows first) in the block to come.
    constexpr int SCALES = (TM + TN + T - 1) / T;
    float next[SCALES];
    auto load_scales = [&](uint32_t kb) {
#pragma unroll
        for (int i = 0; i < SCALES; ++i) {
            const uint32_t r = tid + i * T;
            if (r >= TM + TN) break;
            const bool of_a = r < TM;
            const uint32_t row = of_a ? min(m0 + r, g.m - 1) : min(n0 + r - TM, g.n - 1);
            const uint32_t block = of_a ? g.a_block : g.b_block;
            const int64_t at = static_cast<int64_t>(block == 1 ? row : row / BLOCK_K) * (of_a ? g.sa_pitch : g.sb_pitch) + kb;
            const void* p = of_a ? g.sa : g.sb;
            if constexpr (HARDWARE) {
                next[i] = __uint_as_float(static_cast<const uint8_t*>(p)[at]);
            } else if constexpr (E8M0) {
                next[i] = e8m0_value(static_cast<const uint8_t*>(p)[at]);
            } else {
                next[i] = static_cast<const float*>(p)[at];
            }
        }
    };
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    typedef typename Operand<FAST>::T Frag;
    if (blocks > 0) {
        load_scales(0);
        copy(0);
    }
    for (uint32_t kb = 0; kb < blocks; ++kb) {
        const uint8_t* stage = stages[kb % 2];
        float* sc = scales[kb % 2];
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies and scales have landed
#pragma unroll
        for (int i = 0; i < SCALES; ++i) {
            if (tid + i * T < TM + TN) sc[tid + i * T] = next[i];
        }
        __syncthreads();
        if (kb + 1 < blocks) {
            load_scales(kb + 1);
            copy(kb + 1);
        }
        auto fragment = [&](uint32_t r) {
            const u32x4 lo = *reinterpret_cast<const u32x4*>(stage + r * 128 + ((lane / 16) ^ (r & 7)) * 16);
            const u32x4 hi = *reinterpret_cast<const u32x4*>(stage + r * 128 + ((lane / 16 + 4) ^ (r & 7)) * 16);
            return Frag(lo, hi);
        };
        Frag fa[FM];
        float sa[FM];
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            fa[j] = fragment(wm + 16 * j + lane % 16);
            sa[j] = sc[wm + 16 * j + lane % 16];
        }
        if constexpr (!BROWS && !HARDWARE) {
            const float sb = sc[TM + wn];
#pragma unroll
            for (int j = 0; j < FM; ++j) sa[j] = sa[j] * sb;
        }
        // Row i of fragments: the next one's reads go first, and a product joins its sum LATE products later.
        constexpr int LATE = 2, RING = 4;
        Frag fb[2];
        f32x4 sb[2], p[RING];
        auto read_b = [&](int i) {
            fb[i % 2] = fragment(TM + wn + 16 * i + lane % 16);
            if constexpr (HARDWARE) {
                sb[i % 2][0] = sc[TM + wn + 16 * i + lane % 16];
            } else if constexpr (BROWS) {
                sb[i % 2] = *reinterpret_cast<const f32x4*>(sc + TM + wn + 16 * i + (lane / 16) * 4);
            }
        };
        auto join = [&](int t) {
            const int i = t / FM, j = t % FM;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(BROWS ? sa[j] * sb[i % 2][e] : sa[j], p[t % RING][e], acc[i][j][e]);
        };
        read_b(0);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            if constexpr (!BROWS || HARDWARE) {
                if (i + 1 < FN) read_b(i + 1);
            }
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const int t = i * FM + j;
                if constexpr (HARDWARE) {
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[i % 2].v, fa[j].v, acc[i][j], 0, 0, 0, static_cast<int>(__float_as_uint(sb[i % 2][0])), 0,
                                                                                 static_cast<int>(__float_as_uint(sa[j])));
                } else {
                    if constexpr (FAST) {
                        p[t % RING] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[i % 2].v, fa[j].v, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
                    } else {
                        p[t % RING] = block_product(fb[i % 2], fa[j]);
                    }
                    if (t >= LATE) join(t - LATE);
                }
                if (BROWS && !HARDWARE && j == LATE - 1 && i + 1 < FN) read_b(i + 1);  // the row before has joined
            }
        }
        if constexpr (!HARDWARE) {
#pragma unroll
            for (int t = FM * FN - LATE; t < FM * FN; ++t) join(t);
        }
    }
#pragma unroll
    for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (int j = 0; j < FM; ++j) store_four<OUT>(g, m0 + wm + 16 * j + lane % 16, n0 + wn + 16 * i + (lane / 16) * 4, acc[i][j]);
    }
}

template <uint32_t OUT, bool FAST, bool E8M0, bool BROWS, int TM, int TN, int WM, int WN>
void launch_tile(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    const uint32_t tm = (g.m + TM - 1) / TM, tn = (g.n + TN - 1) / TN;
    hipLaunchKernelGGL((gemm_blocks_tile<OUT, FAST, E8M0, BROWS, TM, TN, WM, WN>), dim3(tm * tn), dim3(WM * WN * 64), 0, s, g, tm, tn);
    launched(ctx, FAST ? "gemm_blocks_fp8" : "gemm_blocks_bf16");
}

bool copies_fit(const GemmBlocksArgs& g) {
    const uint64_t all = reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.b) | static_cast<uint64_t>(g.a_pitch) |
                         static_cast<uint64_t>(g.b_pitch) | g.k;
    return all % 16 == 0 && g.a_pitch < (1 << 23) && g.b_pitch < (1 << 23);
}

template <uint32_t OUT, bool E8M0, int BA, int BB>
void launch_of(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    const uint32_t tm = (g.m + TILE - 1) / TILE, tn = (g.n + TILE - 1) / TILE;
    if (static_cast<uint64_t>(tm) * tn > 0x7fffffffull) fail_invalid("gemm_blocks: too many tiles for one launch");
    hipLaunchKernelGGL((gemm_blocks_any<OUT, E8M0, BA, BB>), dim3(tm * tn), dim3(THREADS), 0, s, g, tm);
    launched(ctx, "gemm_blocks_any");
}

template <uint32_t OUT, bool E8M0>
bool launch_tiles(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    if (!copies_fit(g) || g.m < 64 || g.n < 64) return false;
    if (OUT != LG_DTYPE_F32 && g.k >= 512) {
        if (g.b_block == 1) {
            launch_tile<OUT, true, E8M0, true, 256, 256, 4, 2>(ctx, s, g);
        } else {
            launch_tile<OUT, true, E8M0, false, 256, 256, 4, 2>(ctx, s, g);
        }
    } else if (g.b_block == 1) {
        launch_tile<OUT, false, E8M0, true, 128, 128, 2, 2>(ctx, s, g);
    } else {
        launch_tile<OUT, false, E8M0, false, 128, 128, 2, 2>(ctx, s, g);
    }
    return true;
}

template <uint32_t OUT, bool E8M0>
void launch_blocks(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    if (launch_tiles<OUT, E8M0>(ctx, s, g)) return;
    if (g.a_block == 1 && g.b_block == 1) {
        launch_of<OUT, E8M0, 1, 1>(ctx, s, g);
    } else if (g.a_block == 1) {
        launch_of<OUT, E8M0, 1, 128>(ctx, s, g);
    } else if (g.b_block == 1) {
        launch_of<OUT, E8M0, 128, 1>(ctx, s, g);
    } else {
        launch_of<OUT, E8M0, 128, 128>(ctx, s, g);
    }
}

template <uint32_t OUT>
void launch_out(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    if (g.e8m0) {
        launch_blocks<OUT, true>(ctx, s, g);
    } else {
        launch_blocks<OUT, false>(ctx, s, g);
    }
}

}  // namespace

void launch_gemm_blocks(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    if (g.out == LG_DTYPE_F32) {
        launch_out<LG_DTYPE_F32>(ctx, s, g);
    } else if (g.out == LG_DTYPE_F16) {
        launch_out<LG_DTYPE_F16>(ctx, s, g);
    } else {
        launch_out<LG_DTYPE_BF16>(ctx, s, g);
    }
}

}  // namespace lg
