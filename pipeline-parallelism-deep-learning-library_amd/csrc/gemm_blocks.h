// gfx950 kernels of gemm_blocks: C = alpha * sum over blocks b of sa[m, b] sb[n, b] (A_b . B_b^T) + beta * C
// of e4m3 operands with a scale for each 128 columns of K and each row, or each 128 rows.
//
// The fp8 matrix instructions align each eight neighbouring products to the largest of them and keep 2^-13 of
// it (measured: 1.5e-5 of the norm for normal operands, 1.2e-5 of the sum of absolute products at K = 128).
// Where that is not enough the kernels turn elements into bf16, which holds every e4m3 value, two to an instruction on
// their way to the matrix cores, and multiply on v_mfma_f32_16x16x32_bf16: four of those are a block's sum for 16x16
// outputs, exact products summed in f32 (7e-8 of the norm at K = 4096). The instructions' order of K is free
// as long as both operands share it: a lane takes 32 bytes of one row of each operand (row lane % 16, the
// quarter of the block goes by lane / 16) and eight of them per instruction. B's rows are the first operand and
// A's the second, so a lane's four outputs are neighbours along N of one row of C. A block's sums start
// at zero and join the f32 accumulator by a multiply-add with sa * sb; e8m0 scales are applied by the
// conversion, or are the fp8 instruction's own operands.
#pragma once

#include <algorithm>

#include "head_device.h"

namespace lg {
namespace {

using namespace head_detail;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight e4m3 elements times s, a power of two, as bf16, which holds each of them.
__device__ inline bf16x8 to_bf16(uint32_t lo, uint32_t hi, float s = 1.0f) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's part of a row in a block of 128: 32 elements.
struct Fragment {
    bf16x8 v[4];
    __device__ inline Fragment() {}
    __device__ inline Fragment(u32x4 lo, u32x4 hi, float s = 1.0f) : v{to_bf16(lo[0], lo[1], s), to_bf16(lo[2], lo[3], s), to_bf16(hi[0], hi[1], s), to_bf16(hi[2], hi[3], s)} {}
};

// A block's sums for 16x16 outputs.
__device__ inline f32x4 block_product(const Fragment& b, const Fragment& a, f32x4 p = f32x4{0.0f, 0.0f, 0.0f, 0.0f}) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[i], a.v[i], p, 0, 0, 0);
    return p;
}

__device__ inline float e8m0_value(uint32_t code) {
    // 2^-127, code 0, is subnormal.
    return code == 255 ? __builtin_nanf("") : __uint_as_float(code == 0 ? 0x400000u : code << 23);
}

// Bytes k .. k + 15 of a row of length K at any address, zeros past its end: where they pass it, the row's last sixteen
// shifted down. (Byte by byte under conditions, whose loads the compiler waits for one after another, 77x4099x2011 took 11.9 us
// against 10.2, 1x4099x2011 8.3 against 6.1.)
__device__ inline u32x4 load_sixteen(const uint8_t* row, uint32_t k, uint32_t K) {
    if (k + 16 <= K) return *reinterpret_cast<const u32x4_any*>(row + k);
    u32x4 v = {0, 0, 0, 0};
    if (k >= K) return v;
    if (K < 16) {
#pragma unroll
        for (uint32_t i = 0; i < 15; ++i) {
            const uint32_t byte = row[min(k + i, K - 1)];
            v[i / 4] |= (k + i < K ? byte : 0u) << (8 * (i % 4));
        }
        return v;
    }
    v = *reinterpret_cast<const u32x4_any*>(row + K - 16);
    const uint32_t shift = (k + 16 - K) * 8;  // 8 to 120
    uint64_t lo = v[0] | static_cast<uint64_t>(v[1]) << 32, hi = v[2] | static_cast<uint64_t>(v[3]) << 32;
    lo = shift < 64 ? lo >> shift | hi << (64 - shift) : hi >> (shift - 64);
    hi = shift < 64 ? hi >> shift : 0;
    return u32x4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32)};
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
        __device__ inline T(u32x4 lo, u32x4 hi, float = 1.0f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = static_cast<int>(lo[i]);
                v[i + 4] = static_cast<int>(hi[i]);
            }
        }
    };
};

// Workgroup `id` of `count` to a tile: neighbouring ids go to the eight XCDs in turn, so each XCD takes one
// run of tiles, and runs walk bands of four tiles along M, whose operands its L2 then holds.
__device__ inline void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t* tm, uint32_t* tn) {
    constexpr uint32_t XCDS = 8, BAND = 4;
    const uint32_t count = tiles_m * tiles_n, per = count / XCDS, left = count % XCDS, xcd = id % XCDS;
    const uint32_t t = xcd * per + min(xcd, left) + id / XCDS;
    const uint32_t band = t / (BAND * tiles_n), first = band * BAND, high = min(BAND, tiles_m - first), in = t - first * tiles_n;
    *tm = first + in % high;
    *tn = in / high;
}

// A TM x TN tile of C by KG groups of WM x WN waves. Slices of 128 columns lie in LDS as [row][128] with 16-byte
// chunk c of row r at place c ^ (r & 7), so that eight neighbouring rows' reads of one chunk touch every bank once,
// two stages of KG slices each. DIRECT (bases, pitches and K in whole 16 bytes): copied from memory straight into LDS
// (global_load_lds_dwordx4) while the stage before is multiplied; else through registers, any addresses. Four copies
// go out with each of the first rows of fragments, one row of B's fragments is read ahead, and a product joins its sum
// two products later, so that neither LDS nor the multiply-adds keep the matrix cores waiting. A slice's scales
// pass through registers into LDS beside it. Groups take slices in turn and add their sums in LDS at the end: more
// waves for outputs of few tiles. A group of one wave waits for no other until then.
// FAST multiplies on v_mfma_f32_16x16x128_f8f6f4, one instruction to a block of 16x16 outputs, at the precision
// above; else in bf16.
// Bound by the issue of LDS reads, multiply-adds and matrix instructions of two waves a SIMD; of few tiles by the
// latency of a stage. Measured: 4096x65536x4096 into bf16, f32 scales on 256x256 tiles of eight waves, 1060 us (2080
// TFLOP/s; a library product with one scale 840 us), e8m0 990 us; with rows of C stored by lanes as they hold them 1190 us,
// with bands of eight tiles 1070 us. 8192x8192x4096 into f32 on 128x128 tiles of four waves, two workgroups a compute
// unit: 513 us (1070 TFLOP/s), on 256x128 tiles 517 us; 8192x2048x4096 with e8m0 scales 125 us, multiplied in afterwards
// 155 us. 512x2048x4096 into f32 on 64x64 tiles of two groups 18 us, on 128x128 tiles 40 us; 256x256x4096 on 16x16 tiles of
// sixteen groups 4.9 us, on 32x64 tiles of four 11.9 us. Through registers 77x4099x2011 on 32x64 tiles of four groups 10.2
// us, on 32x32 tiles of eight, whose workgroups are more than the compute units, 14.5 us; 23x7261x1975 10.1 and 8.0 us.
template <uint32_t OUT, bool DIRECT, bool FAST, bool E8M0, bool BROWS, int TM, int TN, int WM, int WN, int KG>
__global__ __launch_bounds__(WM* WN * KG * 64) __attribute__((amdgpu_waves_per_eu(WM * WN * KG > 8 ? WM * WN * KG / 4 : 2))) void gemm_blocks_tile(GemmBlocksArgs g, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int WAVES = WM * WN * KG, T = WAVES * 64, FM = TM / WM / 16, FN = TN / WN / 16;
    constexpr int SLICE = (TM + TN) * 128, STAGE = KG * SLICE, COPIES = STAGE / 16 / T;  // copies a thread; A's rows first
    constexpr int COPIES_A_ROW = 4;                                  // of fragments
    constexpr bool FOLDED = E8M0;  // the operands carry their scales
    static_assert(BROWS || (TN / WN) % 128 == 0 || 128 % (TN / WN) == 0, "a wave's columns share their scale");
    __shared__ __attribute__((aligned(16))) uint8_t stages[2][STAGE];
    __shared__ __attribute__((aligned(16))) float scales[2][KG][TM + TN];  // or e8m0 codes
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const uint32_t kg = wave / (WM * WN);  // the group's slices: kg, kg + KG ...
    uint32_t tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
    const uint32_t m0 = tm * TM, n0 = tn * TN, wm = (wave % WM) * (TM / WM), wn = (wave / WM % WN) * (TN / WN);
    const uint32_t blocks = (g.k + BLOCK_K - 1) / BLOCK_K;
    const uint8_t* pa = g.a + static_cast<int64_t>(m0) * g.a_pitch;
    const uint8_t* pb = g.b + static_cast<int64_t>(n0) * g.b_pitch;
    // Copy i of a wave: 1 KB of a stage, eight rows. Rows past the operand's last one repeat it.
    // Groups of waves copy their own slices.
    constexpr int GW = WM * WN;
    const uint32_t gwave = wave % GW;
    static_assert(TM % (GW * 8) == 0 && TN % (GW * 8) == 0, "a copy is of one operand");
    uint32_t offset[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const uint32_t r = (i * GW + gwave) * 8 + lane / 8, chunk = (lane % 8) ^ (r & 7);
        const bool of_a = i * GW * 8 < TM;
        const uint32_t row = of_a ? min(r, g.m - 1 - m0) : min(r - TM, g.n - 1 - n0);
        offset[i] = row * static_cast<uint32_t>(of_a ? g.a_pitch : g.b_pitch) + chunk * 16;
    }
    u32x4 held[DIRECT ? 1 : COPIES];
    const uint32_t lane_chunk = ((lane % 8) ^ (lane / 8)) * 16;  // of every copy: eight rows at a time
    auto copy = [&](const uint8_t* a, const uint8_t* b, uint32_t at, int i) {
        const uint8_t* from = (i * GW * 8 < TM ? a : b) + offset[i];
        if constexpr (DIRECT) {
            copy_sixteen(from, stages[at] + kg * SLICE + (i * GW + gwave) * 1024);
        } else {
            held[i] = *reinterpret_cast<const u32x4_any*>(from);
        }
    };
    // The start of slice kb of an operand. (The compiler would otherwise keep a 64-bit address for every copy.)
    auto slice = [](const uint8_t* p, uint32_t kb) {
        p += kb * BLOCK_K;
        __asm__("" : "+s"(p));
        return p;
    };
    // Thread t holds the scale of row t of the tile's operands (A's rows first) in the block to come.
    constexpr int SCALES = (TM + TN + GW * 64 - 1) / (GW * 64);
    const uint32_t gtid = tid % (GW * 64);
    float next[SCALES];
    auto load_scales = [&](uint32_t kb) {
#pragma unroll
        for (int i = 0; i < SCALES; ++i) {
            const uint32_t r = gtid + i * GW * 64;
            if (r >= TM + TN) break;
            const bool of_a = r < TM;
            const uint32_t row = of_a ? min(m0 + r, g.m - 1) : min(n0 + r - TM, g.n - 1);
            const uint32_t block = of_a ? g.a_block : g.b_block;
            const int64_t at = static_cast<int64_t>(block == 1 ? row : row / BLOCK_K) * (of_a ? g.sa_pitch : g.sb_pitch) + kb;
            const void* p = of_a ? g.sa : g.sb;
            if constexpr (FAST && E8M0) {
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
    // A product joins its sum LATE products later.
    constexpr int LATE = 2, RING = 4;
    // A fragment's row is lane % 16 past a multiple of 16, so its two chunks' places are the lane's own.
    const uint32_t near = (lane % 16) * 128 + ((lane / 16) ^ (lane & 7)) * 16;
    // Multiplies the slice in stage `at`; `more`: and copies slice kb, a whole one, into the other meanwhile.
    auto multiply = [&](uint32_t at, bool more, uint32_t kb) {
        const uint8_t* rows_a = stages[at] + kg * SLICE + wm * 128;
        const uint8_t* rows_b = stages[at] + kg * SLICE + (TM + wn) * 128;
        const float* sc = scales[at][kg];
        auto fragment = [&](const uint8_t* rows, int i, float scale = 1.0f) {
            const u32x4 lo = *reinterpret_cast<const u32x4*>(rows + near + i * 2048);
            const u32x4 hi = *reinterpret_cast<const u32x4*>(rows + (near ^ 64) + i * 2048);
            return Frag(lo, hi, scale);
        };
        Frag fa[FM], fb[2];
        float sa[FM];
        f32x4 sb[2], p[RING];
        auto read_b = [&](int i) {
            if constexpr (FOLDED) {
                sb[i % 2][0] = sc[TM + wn + 16 * i + lane % 16];
            } else if constexpr (BROWS) {
                sb[i % 2] = *reinterpret_cast<const f32x4*>(sc + TM + wn + 16 * i + (lane / 16) * 4);
            }
            fb[i % 2] = fragment(rows_b, i, FOLDED ? sb[i % 2][0] : 1.0f);
        };
        auto join = [&](int t) {
            const int i = t / FM, j = t % FM;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(BROWS ? sa[j] * sb[i % 2][e] : sa[j], p[t % RING][e], acc[i][j][e]);
        };
        read_b(0);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            sa[j] = sc[wm + 16 * j + lane % 16];
            fa[j] = fragment(rows_a, j, FOLDED ? sa[j] : 1.0f);
        }
        if constexpr (!BROWS && !FOLDED) {
            const float b = sc[TM + wn];
#pragma unroll
            for (int j = 0; j < FM; ++j) sa[j] = sa[j] * b;
        }
        if (more) load_scales(kb);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            if constexpr (!BROWS || FOLDED) {
                if (i + 1 < FN) read_b(i + 1);
            }
            if (more && i * COPIES_A_ROW < COPIES) {
                const uint8_t *ca = slice(pa, kb), *cb = slice(pb, kb);
#pragma unroll
                for (int q = 0; q < COPIES_A_ROW; ++q) {
                    if (i * COPIES_A_ROW + q < COPIES) copy(ca, cb, at ^ 1, i * COPIES_A_ROW + q);
                }
            }
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const int t = i * FM + j;
                if constexpr (FOLDED && !FAST) {
                    acc[i][j] = block_product(fb[i % 2], fa[j], acc[i][j]);
                } else if constexpr (FOLDED) {
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
                if (BROWS && !FOLDED && j == LATE - 1 && i + 1 < FN) read_b(i + 1);  // the row before has joined
            }
            if constexpr (!FAST) {
#pragma unroll
                for (int j = 0; j < 4 * FM; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (j < 2) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < FM; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (j < 2) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    if (!FOLDED) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!FOLDED) {
#pragma unroll
            for (int t = FM * FN - LATE; t < FM * FN; ++t) join(t);
        }
    };
    // The last slice, which may be of fewer than 128 columns, goes first, with zeros in the places past them; then the
    // others in order: turn q of group kg is slice q * KG + kg - 1.
    const uint32_t turns = (blocks + KG - 1) / KG;
    if (kg < blocks) {
        const uint32_t kb = kg == 0 ? blocks - 1 : kg - 1;
        load_scales(kb);
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            if constexpr (DIRECT) {
                if (kb * BLOCK_K + lane_chunk < g.k) {
                    copy(slice(pa, kb), slice(pb, kb), 0, i);
                } else {
                    *reinterpret_cast<u32x4*>(stages[0] + kg * SLICE + (i * GW + gwave) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
                }
            } else if ((kb + 1) * BLOCK_K <= g.k) {
                copy(slice(pa, kb), slice(pb, kb), 0, i);
            } else {
                held[i] = load_sixteen((i * GW * 8 < TM ? pa : pb) + (offset[i] - lane_chunk), kb * BLOCK_K + lane_chunk, g.k);
            }
        }
    }
    for (uint32_t s = 0; s < turns; ++s) {
        const bool live = s * KG + kg < blocks;
        float* sc = scales[s % 2][kg];
        if (live) {
            if constexpr (DIRECT) {
                __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies and scales have landed
            } else {
#pragma unroll
                for (int i = 0; i < COPIES; ++i) *reinterpret_cast<u32x4*>(stages[s % 2] + kg * SLICE + (i * GW + gwave) * 1024 + lane * 16) = held[i];
            }
#pragma unroll
            for (int i = 0; i < SCALES; ++i) {
                if (gtid + i * GW * 64 < TM + TN) sc[gtid + i * GW * 64] = next[i];
            }
        }
        if constexpr (GW > 1) {
            __syncthreads();
        } else {
            __asm__ volatile("" ::: "memory");  // a group of one wave reads its own slices only
        }
        if (live) multiply(s % 2, (s + 1) * KG + kg < blocks, (s + 1) * KG + kg - 1);
    }
    if constexpr (KG > 1) {
        // The groups' sums meet in LDS, in their order.
        constexpr int SUMS = FM * FN * 1024;  // bytes of a wave
        static_assert((KG - 1) * GW * SUMS <= 2 * STAGE, "the groups' sums fit the stages");
        uint8_t* sums = &stages[0][0];
        __syncthreads();
        if (kg > 0) {
#pragma unroll
            for (int i = 0; i < FN * FM; ++i) *reinterpret_cast<f32x4*>(sums + ((kg - 1) * GW + gwave) * SUMS + i * 1024 + lane * 16) = acc[i / FM][i % FM];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int o = 0; o < KG - 1; ++o) {
#pragma unroll
            for (int i = 0; i < FN * FM; ++i) acc[i / FM][i % FM] = acc[i / FM][i % FM] + *reinterpret_cast<const f32x4*>(sums + (o * GW + gwave) * SUMS + i * 1024 + lane * 16);
        }
    }
    constexpr int ROW = TN / WN * static_cast<int>(elem_size<OUT>), CHUNKS = ROW / 16, PER = 16 / static_cast<int>(elem_size<OUT>);
    constexpr bool WHOLE = KG == 1 && (CHUNKS == 8 || CHUNKS == 16) && TM / WM * ROW * WAVES <= 2 * STAGE;
    if (!WHOLE || g.beta != 0.0f) {
#pragma unroll
        for (int i = 0; i < FN; ++i) {
#pragma unroll
            for (int j = 0; j < FM; ++j) store_four<OUT>(g, m0 + wm + 16 * j + lane % 16, n0 + wn + 16 * i + (lane / 16) * 4, acc[i][j]);
        }
        return;
    }
    if constexpr (WHOLE) {
    // A wave's outputs pass through its own part of the stages, so that rows leave as whole runs of 16 bytes a lane:
    // [row][16-byte chunk], chunk c of row r at place c ^ (r % CHUNKS).
    __syncthreads();  // every wave is done with the stages
    uint8_t* mine = &stages[0][0] + wave * (TM / WM * ROW);
#pragma unroll
    for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const uint32_t r = 16 * j + lane % 16, byte = (16 * i + (lane / 16) * 4) * elem_size<OUT>;
            uint8_t* to = mine + r * ROW + (((byte / 16) ^ (r % CHUNKS)) * 16 + byte % 16);
            const f32x4 v = acc[i][j] * g.alpha;
            if constexpr (OUT == LG_DTYPE_F32) {
                *reinterpret_cast<f32x4*>(to) = v;
            } else {
                *reinterpret_cast<u32x2*>(to) = u32x2{pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3])};
            }
        }
    }
    // The wave's own writes only: no other wave reads them.
    __builtin_amdgcn_wave_barrier();
    const uint32_t c = lane % CHUNKS, n = n0 + wn + c * PER;
#pragma unroll
    for (int q = 0; q < TM / WM * CHUNKS / 64; ++q) {
        const uint32_t r = q * (64 / CHUNKS) + lane / CHUNKS, m = m0 + wm + r;
        const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * ROW + (c ^ (r % CHUNKS)) * 16);
        if (m >= g.m || n >= g.n) continue;
        char* to = static_cast<char*>(g.c) + (m * g.c_pitch + n) * elem_size<OUT>;
        if (n + PER <= g.n) {
            *reinterpret_cast<u32x4_any*>(to) = v;
        } else {
            for (uint32_t e = 0; n + e < g.n; ++e) {
                if constexpr (OUT == LG_DTYPE_F32) {
                    reinterpret_cast<uint32_t*>(to)[e] = v[e];
                } else {
                    reinterpret_cast<uint16_t*>(to)[e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e % 2)));
                }
            }
        }
    }
    }
}

template <uint32_t OUT, bool DIRECT, bool FAST, bool E8M0, bool BROWS, int TM, int TN, int WM, int WN, int KG>
void launch_tile(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g, const char* name) {
    const uint32_t tm = (g.m + TM - 1) / TM, tn = (g.n + TN - 1) / TN;
    hipLaunchKernelGGL((gemm_blocks_tile<OUT, DIRECT, FAST, E8M0, BROWS, TM, TN, WM, WN, KG>), dim3(tm * tn), dim3(WM * WN * KG * 64), 0, s, g, tm, tn);
    launched(ctx, name);
}

// Few rows of A, at any address: a workgroup takes 32 rows of B and 16 of A, its four waves equal runs of
// blocks, whose sums meet in LDS in the waves' order. Each byte of B goes from memory into the registers of the one
// wave that multiplies it, 32 consecutive bytes a lane, the next block's while this one's is multiplied. A lane reads a row
// of its own, of which the caches serve a compute unit sixteen bytes a cycle: enough where every compute unit reads
// (then bound by reading B: 1x65536x4096 46.6 us, 5.8 TB/s; 38.7 us of weights that the last call left in the caches),
// too little where few do (1x4096x4096 7.3 us, on 16x16 tiles 4.7).
template <uint32_t OUT, bool E8M0, bool BROWS, int FN, int W>
__global__ __launch_bounds__(W * 64) void gemm_blocks_thin(GemmBlocksArgs g, uint32_t tiles_n) {
    __shared__ f32x4 sums[W][FN][64];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const uint32_t n0 = (blockIdx.x % tiles_n) * 16 * FN, m0 = (blockIdx.x / tiles_n) * 16;
    const uint32_t blocks = (g.k + BLOCK_K - 1) / BLOCK_K, per = (blocks + W - 1) / W;
    const uint32_t lo = min(wave * per, blocks), hi = min(lo + per, blocks);
    const uint32_t row = lane % 16, part = (lane / 16) * 32;
    const uint8_t* pb[FN];
    const char* psb[FN][BROWS && !E8M0 ? 4 : 1];
    constexpr int SIZE = E8M0 ? 1 : 4;
    const uint32_t m = min(m0 + row, g.m - 1);
    const uint8_t* pa = g.a + m * g.a_pitch + part;
    const char* psa = static_cast<const char*>(g.sa) + (g.a_block == 1 ? m : m / BLOCK_K) * g.sa_pitch * SIZE;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const uint32_t n = min(n0 + 16 * i + row, g.n - 1);
        pb[i] = g.b + n * g.b_pitch + part;
        // e8m0 scales go with the lane's row of B, f32 ones with its four outputs' columns.
        if constexpr (E8M0) {
            psb[i][0] = static_cast<const char*>(g.sb) + (g.b_block == 1 ? n : n / BLOCK_K) * g.sb_pitch;
        } else if constexpr (BROWS) {
#pragma unroll
            for (int e = 0; e < 4; ++e) psb[i][e] = static_cast<const char*>(g.sb) + min(n0 + 16 * i + (lane / 16) * 4 + e, g.n - 1) * g.sb_pitch * 4;
        } else {
            psb[i][0] = static_cast<const char*>(g.sb) + ((n0 + 16 * i) / BLOCK_K) * g.sb_pitch * 4;
        }
    }
    f32x4 acc[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    struct Slice {
        u32x4 a[2], b[FN][2];
        float sa, sb[FN][BROWS && !E8M0 ? 4 : 1];
    };
    auto load = [&](uint32_t kb, Slice& s) {
        const uint32_t k = kb * BLOCK_K;
        if (k + BLOCK_K <= g.k) {
#pragma unroll
            for (int i = 0; i < FN; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) s.b[i][h] = *reinterpret_cast<const u32x4_any*>(pb[i] + k + 16 * h);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) s.a[h] = *reinterpret_cast<const u32x4_any*>(pa + k + 16 * h);
        } else {
            for (int h = 0; h < 2; ++h) {
                for (int i = 0; i < FN; ++i) s.b[i][h] = load_sixteen(pb[i] - part, k + part + 16 * h, g.k);
                s.a[h] = load_sixteen(pa - part, k + part + 16 * h, g.k);
            }
        }
        auto scale = [&](const char* p) { return E8M0 ? e8m0_value(reinterpret_cast<const uint8_t*>(p)[kb]) : reinterpret_cast<const float*>(p)[kb]; };
        s.sa = scale(psa);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
#pragma unroll
            for (int e = 0; e < (BROWS && !E8M0 ? 4 : 1); ++e) s.sb[i][e] = scale(psb[i][e]);
        }
    };
    auto multiply = [&](const Slice& s) {
        const Fragment fa(s.a[0], s.a[1], E8M0 ? s.sa : 1.0f);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const Fragment fb(s.b[i][0], s.b[i][1], E8M0 ? s.sb[i][0] : 1.0f);
            if constexpr (E8M0) {
                acc[i] = block_product(fb, fa, acc[i]);
            } else {
                const f32x4 p = block_product(fb, fa);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = __builtin_fmaf(s.sa * s.sb[i][BROWS ? e : 0], p[e], acc[i][e]);
            }
        }
    };
    if (lo < hi) {
        Slice s[2];
        load(lo, s[0]);
        for (uint32_t kb = lo; kb < hi; kb += 2) {
            if (kb + 1 < hi) load(kb + 1, s[1]);
            multiply(s[0]);
            if (kb + 1 >= hi) break;
            if (kb + 2 < hi) load(kb + 2, s[0]);
            multiply(s[1]);
        }
    }
#pragma unroll
    for (int i = 0; i < FN; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int q = wave; q < FN; q += W) {
        f32x4 v = sums[0][q][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v = v + sums[w][q][lane];
        store_four<OUT>(g, m0 + lane % 16, n0 + 16 * q + (lane / 16) * 4, v);
    }
}

template <uint32_t OUT, bool E8M0, bool BROWS, int FN, int W>
void launch_thin(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    const uint32_t tm = (g.m + 15) / 16, tn = (g.n + 16 * FN - 1) / (16 * FN);
    hipLaunchKernelGGL((gemm_blocks_thin<OUT, E8M0, BROWS, FN, W>), dim3(tm * tn), dim3(W * 64), 0, s, g, tn);
    launched(ctx, "gemm_blocks_thin");
}

bool copies_fit(const GemmBlocksArgs& g) {
    const uint64_t all = reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.b) | static_cast<uint64_t>(g.a_pitch) |
                         static_cast<uint64_t>(g.b_pitch) | g.k;
    return all % 16 == 0;
}

// Which kernel is fastest is told by a model of its time: rounds of workgroups over the 256 compute units, each round a fixed
// part and one for every turn of its groups along K. The figures, in hundredths of a microsecond, are a fit over 320
// products with sizes spread evenly over the logarithms of 1 to 8192 rows, 128 to 16384 columns and K of 200 to 8192, each
// timed on every kernel: the kernel with the least modelled time took 1.04 times the time of the fastest on
// average. `share`: workgroups that share a compute unit, from 257 tiles on; 0: many, without rounds.
struct Cost {
    uint32_t m, n, groups, share;
    struct {
        uint32_t fixed, turn, shared_fixed, shared_turn;
    } any, direct;  // through registers, timed at odd pitches; copied straight into LDS
};
enum Plan { THIN, BF16_128, BF16_64, BF16_32X64, BF16_32, BF16_16, FP8_256, FP8_128, FP8_64, FP8_32X64, FP8_32, PLANS };
constexpr Cost COSTS[PLANS] = {
    {16, 32, 4, 0, {76, 142, 0, 120}, {71, 55, 15, 50}},
    {128, 128, 1, 2, {246, 133, 309, 314}, {177, 115, 314, 192}},
    {64, 64, 2, 2, {134, 128, 270, 187}, {75, 88, 152, 145}},
    {32, 64, 4, 1, {138, 157, 0, 0}, {107, 105, 0, 0}},
    {32, 32, 8, 1, {134, 187, 0, 0}, {95, 113, 0, 0}},
    {16, 16, 16, 1, {117, 160, 0, 0}, {78, 96, 0, 0}},
    {256, 256, 1, 1, {0, 0, 0, 0}, {322, 150, 0, 0}},
    {128, 128, 1, 2, {86, 122, 454, 187}, {155, 71, 227, 129}},
    {64, 64, 2, 2, {92, 118, 120, 180}, {85, 58, 118, 113}},
    {32, 64, 4, 1, {51, 164, 0, 0}, {97, 78, 0, 0}},
    {32, 32, 8, 1, {136, 176, 0, 0}, {103, 87, 0, 0}},
};
inline Plan plan_of(const GemmBlocksArgs& g, bool direct) {
    // Pitches from 2^23 on would pass 32 bits within a tile.
    if (g.a_pitch >= (1 << 23) || g.b_pitch >= (1 << 23)) return THIN;
    // The fp8 instruction's precision is enough for 16-bit outputs of long sums.
    const bool fast = g.out != LG_DTYPE_F32 && g.k >= 512;
    auto time = [&](int p) {
        const Cost& c = COSTS[p];
        const auto& t = direct ? c.direct : c.any;
        const uint64_t tiles = static_cast<uint64_t>((g.m + c.m - 1) / c.m) * ((g.n + c.n - 1) / c.n);
        const uint64_t turns = ((g.k + BLOCK_K - 1) / BLOCK_K + c.groups - 1) / c.groups;
        if (c.share == 0 && tiles > 256) return tiles * (t.shared_fixed + t.shared_turn * turns) / 256;
        return c.share <= 1 || tiles <= 256 ? (tiles + 255) / 256 * (t.fixed + t.turn * turns)
                                              : (tiles + 256 * c.share - 1) / (256 * c.share) * (t.shared_fixed + t.shared_turn * turns);
    };
    Plan plan = BF16_128;
    uint64_t best = time(plan);
    for (int p = BF16_64; p < (fast ? PLANS : FP8_256); ++p) {
        if (p == FP8_256 && !direct) continue;
        if (const uint64_t t = time(p); t < best) {
            best = t;
            plan = static_cast<Plan>(p);
        }
    }
    // Tiles read B at 4.8 TB/s at the best (1x65536x4096 53 us, THIN 39 us; 1x32000x2048 16.7 and 13.2 us).
    const uint64_t reading = static_cast<uint64_t>(g.n) * g.k / 48000;
    return g.m <= 16 && time(THIN) <= std::max(best, reading) ? THIN : plan;
}

template <uint32_t OUT, bool DIRECT, bool E8M0, bool BROWS>
void launch_of(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    const Plan plan = plan_of(g, DIRECT);
    if constexpr (OUT != LG_DTYPE_F32) {
        switch (plan) {
            case FP8_256:
                if constexpr (DIRECT) launch_tile<OUT, true, true, E8M0, BROWS, 256, 256, 4, 2, 1>(ctx, s, g, "gemm_blocks_fp8_256x256");
                return;
            case FP8_128:
                return launch_tile<OUT, DIRECT, true, E8M0, BROWS, 128, 128, DIRECT ? 2 : 4, 2, 1>(ctx, s, g, DIRECT ? "gemm_blocks_fp8_128x128" : "gemm_blocks_fp8_128x128_any");
            case FP8_64:
                return launch_tile<OUT, DIRECT, true, E8M0, BROWS, 64, 64, 2, 2, 2>(ctx, s, g, DIRECT ? "gemm_blocks_fp8_64x64" : "gemm_blocks_fp8_64x64_any");
            case FP8_32X64:
                return launch_tile<OUT, DIRECT, true, E8M0, BROWS, 32, 64, 1, 4, 4>(ctx, s, g, DIRECT ? "gemm_blocks_fp8_32x64" : "gemm_blocks_fp8_32x64_any");
            case FP8_32:
                return launch_tile<OUT, DIRECT, true, E8M0, BROWS, 32, 32, 1, 2, 8>(ctx, s, g, DIRECT ? "gemm_blocks_fp8_32x32" : "gemm_blocks_fp8_32x32_any");
            default:
                break;
        }
    }
    switch (plan) {
        case BF16_128:
            return launch_tile<OUT, DIRECT, false, E8M0, BROWS, 128, 128, DIRECT ? 2 : 4, 2, 1>(ctx, s, g, DIRECT ? "gemm_blocks_bf16_128x128" : "gemm_blocks_bf16_128x128_any");
        case BF16_64:
            return launch_tile<OUT, DIRECT, false, E8M0, BROWS, 64, 64, 2, 2, 2>(ctx, s, g, DIRECT ? "gemm_blocks_bf16_64x64" : "gemm_blocks_bf16_64x64_any");
        case BF16_32X64:
            return launch_tile<OUT, DIRECT, false, E8M0, BROWS, 32, 64, 1, 4, 4>(ctx, s, g, DIRECT ? "gemm_blocks_bf16_32x64" : "gemm_blocks_bf16_32x64_any");
        case BF16_32:
            return launch_tile<OUT, DIRECT, false, E8M0, BROWS, 32, 32, 1, 2, 8>(ctx, s, g, DIRECT ? "gemm_blocks_bf16_32x32" : "gemm_blocks_bf16_32x32_any");
        case BF16_16:
            return launch_tile<OUT, DIRECT, false, E8M0, BROWS, 16, 16, 1, 1, 16>(ctx, s, g, DIRECT ? "gemm_blocks_bf16_16x16" : "gemm_blocks_bf16_16x16_any");
        default:
            return launch_thin<OUT, E8M0, BROWS, 2, 4>(ctx, s, g);
    }
}

template <uint32_t OUT, bool E8M0, bool BROWS>
void launch_at(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    copies_fit(g) ? launch_of<OUT, true, E8M0, BROWS>(ctx, s, g) : launch_of<OUT, false, E8M0, BROWS>(ctx, s, g);
}

}  // namespace

template <uint32_t OUT>
void launch_gemm_blocks_into(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    if (g.e8m0) {
        launch_at<OUT, true, true>(ctx, s, g);
    } else if (g.b_block == 1) {
        launch_at<OUT, false, true>(ctx, s, g);
    } else {
        launch_at<OUT, false, false>(ctx, s, g);
    }
}

}  // namespace lg
