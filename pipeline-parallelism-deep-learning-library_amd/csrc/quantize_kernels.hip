// gfx950 kernels of quantize_blocks: e4m3 elements with a scale for each block of 128 columns and one
// or 128 rows.
//
// A block's largest magnitude A is the integer maximum of the elements' bits without the sign, which
// orders infinities and NaNs above every number; it counts as 2^-100 at the least, so neither the scale
// nor its inverse leaves f32's normal range. f32 scales: s = A / 448 and inv = 448 / A, each rounded
// once; e8m0 scales: s = 2^e, the smallest power of two with A <= 448 s, whose inverse is exact, so that
// every element of a 16-bit or f32 matrix is rounded once. q = x * inv rounded to e4m3, to nearest,
// ties to even (v_cvt_pk_fp8_f32); |x| * inv rounds to 448 at the most, so nothing overflows.
#include <algorithm>

#include "head_device.h"

namespace lg {
namespace {

using namespace head_detail;

constexpr int THREADS = 256;
constexpr int GROUP_LANES = 16;  // lanes that hold a block's row of 128, eight elements each
constexpr float SMALLEST = 0x1p-100f;
constexpr uint32_t INF = 0x7f800000u;

__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The scale of a block whose largest magnitude has the bits `top`, and its inverse.
template <bool E8M0>
struct Scale {
    float inverse;
    float value;    // f32 scales
    uint8_t code;   // e8m0 scales
    __device__ inline explicit Scale(uint32_t top) {
        const bool finite = top < INF;
        const float a = fmaxf(__uint_as_float(top), SMALLEST);
        if constexpr (E8M0) {
            // 448 = 1.75 * 2^8: a <= 448 * 2^e from e = exponent(a) - 8, one more where the significand passes 1.75.
            const uint32_t bits = __float_as_uint(a);
            const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
            inverse = finite ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) : __builtin_nanf("");
            code = finite ? static_cast<uint8_t>(e + 127) : 255;
        } else {
            value = finite ? a / 448.0f : __builtin_nanf("");
            inverse = finite ? 448.0f / a : __builtin_nanf("");
        }
    }
    __device__ inline void store(void* s, int64_t at) const {
        if constexpr (E8M0) {
            static_cast<uint8_t*>(s)[at] = code;
        } else {
            static_cast<float*>(s)[at] = value;
        }
    }
};

// Eight elements times `inverse` as e4m3.
__device__ inline u32x2 to_e4m3(const float (&v)[8], float inverse) {
    u32x2 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inverse, v[4 * i + 1] * inverse, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inverse, v[4 * i + 3] * inverse, w, true);
        o[i] = static_cast<uint32_t>(w);
    }
    return o;
}

// Columns c .. c + 7 of a row of `cols` at p, zeros past its end, where the last column is read instead: loads without
// branches go out together (16383x1023 bf16 transposed 15.4 us, with a load under each condition 20.6).
template <uint32_t DT>
__device__ inline void load_eight(const char* p, uint32_t c, uint32_t cols, float (&v)[8]) {
    if (c + 8 <= cols) {
        Run<DT> r;
        r.load(p + static_cast<uint64_t>(c) * elem_size<DT>);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r[e];
    } else if (c >= cols) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float w = load_one<DT>(p + static_cast<uint64_t>(min(c + e, cols - 1)) * elem_size<DT>);
            v[e] = c + e < cols ? w : 0.0f;
        }
    }
}

// The same of two runs of four, 64 columns apart.
template <uint32_t DT>
__device__ inline void load_halves(const char* p, uint32_t c, uint32_t cols, float (&v)[8]) {
    static_assert(DT == LG_DTYPE_F32, "a lane's 16 bytes are four elements");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = c + 64 * h;
        if (at + 4 <= cols) {
            const u32x4 w = *reinterpret_cast<const u32x4_any*>(p + static_cast<uint64_t>(at) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * h + e] = __uint_as_float(w[e]);
        } else if (at >= cols) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * h + e] = 0.0f;
} else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * h + e] = at + e < cols ? load_one<DT>(p + static_cast<uint64_t>(at + e) * 4) : 0.0f;
        }
    }
}

__device__ inline void store_eight(uint8_t* row, uint32_t c, uint32_t cols, u32x2 o) {
    if (c + 8 <= cols) {
        *reinterpret_cast<u32x2_any*>(row + c) = o;
    } else {
        for (uint32_t e = 0; c + e < cols && e < 8; ++e) row[c + e] = static_cast<uint8_t>(o[e / 4] >> (8 * (e % 4)));
    }
}

// A scale for each row: sixteen lanes take a row's 128 columns; the maximum passes between them. One read and one write of
// everything, bound by memory: 4096x16384 bf16 38.7 us (5.2 TB/s, a large copy's rate); one row of 4096 3.4 us, a launch.
template <uint32_t DT, bool E8M0>
__global__ __launch_bounds__(THREADS) void quantize_rows(QuantizeArgs a, uint32_t groups) {
    const uint64_t group = (static_cast<uint64_t>(blockIdx.x) * THREADS + threadIdx.x) / GROUP_LANES;
    if (group >= static_cast<uint64_t>(a.rows) * groups) return;  // whole groups of lanes at once
    const uint32_t row = static_cast<uint32_t>(group / groups), g = static_cast<uint32_t>(group % groups);
    const uint32_t lane = threadIdx.x % GROUP_LANES, c = g * BLOCK_K + lane * 8;
    float v[8];
    load_eight<DT>(static_cast<const char*>(a.x) + row * a.x_pitch * elem_size<DT>, c, a.cols, v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
#pragma unroll
    for (int d = 1; d < GROUP_LANES; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, GROUP_LANES)));
    const Scale<E8M0> s(top);
    store_eight(a.q + row * a.q_pitch, c, a.cols, to_e4m3(v, s.inverse));
    if (lane == 0) s.store(a.s, row * a.s_pitch + g);
}

// A 128x128 tile of q by 256 threads: thread t holds eight runs of eight elements along the axis that is contiguous in x
// (of f32 two runs of four for T, so that a load of sixteen lanes is 256 bytes in a row). T: that axis is q's rows, and
// the tile turns in LDS, [row][128] with 8-byte run l of row r at place l ^ (r / 8), so that q's rows leave in whole runs
// of 128 bytes. Neighbouring tiles of a row of them go to one XCD, whose L2 then joins the lines that two tiles share;
// `in_turn`: to the XCDs in turn, which is faster for tiles that lie as x does and share no lines (4096x16384 bf16 43.8 us
// against 51.9; 3000x20000 49.1 against 40.5). Bound by memory, and at odd pitches by the lines that tiles read and write
// in part: 8191x4099 f32 transposed 40.3 us (4.2 TB/s); by lanes that store what they hold, without LDS, 51 us,
// neighbours on different XCDs 44 us.
constexpr int TILE = 128;

template <uint32_t DT, bool E8M0, bool T, bool BLOCK>
__global__ __launch_bounds__(THREADS) void quantize_tile(QuantizeArgs a, uint32_t tiles_c, bool in_turn) {
    static_assert(T || BLOCK, "rows of their own scales are quantize_rows'");
    constexpr uint32_t XCDS = 8;
    const uint32_t per = gridDim.x / XCDS, left = gridDim.x % XCDS, xcd = blockIdx.x % XCDS;
    const uint32_t tile = in_turn ? blockIdx.x : xcd * per + min(xcd, left) + blockIdx.x / XCDS, tr = tile / tiles_c, tc = tile % tiles_c;
    const uint32_t r0 = tr * TILE, c0 = tc * TILE, tid = threadIdx.x;
    const uint32_t along = tid % 16, line = tid / 16;
    constexpr bool HALVES = T && DT == LG_DTYPE_F32;
    auto row_of = [&](int e) { return HALVES ? 4 * along + e % 4 + 64 * (e / 4) : 8 * along + e; };  // T: element e's, in the tile
    // Run i, T: column c0 + 8 line + i, rows r0 + 8 along ...; else row r0 + line + 16 i, columns c0 + 8 along ...
    float v[8][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t l = T ? c0 + 8 * line + i : r0 + line + 16 * i;
        if (l < (T ? a.cols : a.rows)) {
            const char* p = static_cast<const char*>(a.x) + l * a.x_pitch * elem_size<DT>;
            if constexpr (HALVES) {
                load_halves<DT>(p, r0 + 4 * along, a.rows, v[i]);
            } else {
                load_eight<DT>(p, (T ? r0 : c0) + 8 * along, T ? a.rows : a.cols, v[i]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        }
    }
    float inverse[BLOCK ? 1 : 8];
    if constexpr (BLOCK) {
        __shared__ uint32_t tops[THREADS / 64];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[i][e]));
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
        if (tid % 64 == 0) tops[tid / 64] = top;
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        const Scale<E8M0> s(top);
        if (tid == 0) s.store(a.s, tr * a.s_pitch + tc);
        inverse[0] = s.inverse;
    } else {
        // A scale for each of the tile's rows: the sixteen lines' maxima of a row meet in LDS.
        __shared__ uint32_t tops[16][TILE];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i][e]));
            tops[line][row_of(e)] = m;
        }
        __syncthreads();
        __shared__ float inverses[TILE];
        if (tid < TILE) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, tops[i][tid]);
            const Scale<E8M0> s(m);
            inverses[tid] = s.inverse;
            if (r0 + tid < a.rows) s.store(a.s, (r0 + tid) * a.s_pitch + tc);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) inverse[e] = inverses[row_of(e)];
    }
    if constexpr (!T) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t r = r0 + line + 16 * i;
            if (r < a.rows) store_eight(a.q + r * a.q_pitch, c0 + 8 * along, a.cols, to_e4m3(v[i], inverse[0]));
        }
    } else {
        __shared__ u32x2 turned[TILE][16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float w[8] = {v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
            turned[row_of(e)][line ^ (row_of(e) / 8)] = to_e4m3(w, inverse[BLOCK ? 0 : e]);
        }
        __syncthreads();
        const uint32_t chunk = tid % 8, c = c0 + 16 * chunk;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t l = tid / 8 + 32 * i, r = r0 + l;
            if (r >= a.rows) break;
            const u32x2 lo = turned[l][(2 * chunk) ^ (l / 8)], hi = turned[l][(2 * chunk + 1) ^ (l / 8)];
            uint8_t* row = a.q + r * a.q_pitch;
            if (c + 16 <= a.cols) {
                *reinterpret_cast<u32x4_any*>(row + c) = u32x4{lo[0], lo[1], hi[0], hi[1]};
            } else {
                store_eight(row, c, a.cols, lo);
                store_eight(row, c + 8, a.cols, hi);
            }
        }
    }
}

template <uint32_t DT, bool E8M0>
void launch_of(Context* ctx, hipStream_t s, const QuantizeArgs& a) {
    const uint32_t groups = (a.cols + BLOCK_K - 1) / BLOCK_K, bands = (a.rows + TILE - 1) / TILE;
    if (a.block == 1 && !a.transposed) {
        // A launch's threads have 32-bit numbers: rows beyond them go in launches of their own.
        const uint64_t most = (1ull << 31) / (static_cast<uint64_t>(groups) * GROUP_LANES);
        for (uint64_t r = 0; r < a.rows; r += most) {
            QuantizeArgs p = a;
            p.rows = static_cast<uint32_t>(a.rows - r < most ? a.rows - r : most);
            p.x = static_cast<const char*>(a.x) + static_cast<int64_t>(r) * a.x_pitch * elem_size<DT>;
            p.q = a.q + static_cast<int64_t>(r) * a.q_pitch;
            p.s = static_cast<char*>(a.s) + static_cast<int64_t>(r) * a.s_pitch * (E8M0 ? 1 : 4);
            const uint64_t wgs = (static_cast<uint64_t>(p.rows) * groups * GROUP_LANES + THREADS - 1) / THREADS;
            hipLaunchKernelGGL((quantize_rows<DT, E8M0>), dim3(static_cast<uint32_t>(wgs)), dim3(THREADS), 0, s, p, groups);
            launched(ctx, "quantize_rows");
        }
        return;
    }
    const uint64_t places = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.q) | static_cast<uint64_t>(a.x_pitch * elem_size<DT>) | static_cast<uint64_t>(a.q_pitch);
    const bool whole_lines = places % 128 == 0;
    // So do bands of 128 rows. (Rows have at most 2^29 columns, 2^22 groups.)
    const uint32_t most = (1u << 23) / groups;
    for (uint32_t b = 0; b < bands; b += most) {
        QuantizeArgs p = a;
        const int64_t row = static_cast<int64_t>(b) * TILE;
        const uint32_t n = std::min(bands - b, most);
        p.rows = static_cast<uint32_t>(std::min<int64_t>(a.rows - row, static_cast<int64_t>(n) * TILE));
        p.x = static_cast<const char*>(a.x) + row * (a.transposed ? 1 : a.x_pitch) * elem_size<DT>;
        p.q = a.q + row * a.q_pitch;
        p.s = static_cast<char*>(a.s) + (a.block == 1 ? row : b) * a.s_pitch * (E8M0 ? 1 : 4);
        const dim3 grid(n * groups), threads(THREADS);
        if (a.block == 1) {
            hipLaunchKernelGGL((quantize_tile<DT, E8M0, true, false>), grid, threads, 0, s, p, groups, false);
            launched(ctx, "quantize_rows_t");
        } else if (a.transposed) {
            hipLaunchKernelGGL((quantize_tile<DT, E8M0, true, true>), grid, threads, 0, s, p, groups, false);
            launched(ctx, "quantize_tiles_t");
        } else {
            hipLaunchKernelGGL((quantize_tile<DT, E8M0, false, true>), grid, threads, 0, s, p, groups, whole_lines);
            launched(ctx, "quantize_tiles");
        }
    }
}

template <uint32_t DT>
void launch_dtype(Context* ctx, hipStream_t s, const QuantizeArgs& a) {
    if (a.e8m0) {
        launch_of<DT, true>(ctx, s, a);
    } else {
        launch_of<DT, false>(ctx, s, a);
    }
}

}  // namespace

void launch_quantize_blocks(Context* ctx, hipStream_t s, const QuantizeArgs& a) {
    if (a.dtype == LG_DTYPE_F32) {
        launch_dtype<LG_DTYPE_F32>(ctx, s, a);
    } else if (a.dtype == LG_DTYPE_F16) {
        launch_dtype<LG_DTYPE_F16>(ctx, s, a);
    } else {
        launch_dtype<LG_DTYPE_BF16>(ctx, s, a);
    }
}

}  // namespace lg
