// gfx950 kernels over rows of logits: log probabilities with entropy and top alternatives, their
// gradient, and distillation's loss and gradient.
//
// One pass reads a row once: each thread keeps a running maximum m and, relative to it, s = sum of
// 2^d and u = sum of 2^d d with d = (x - m) log2(e) / T, rescaled when m grows; sums of eight elements
// are f32, everything above them f64, so a row whose probability lies on one element keeps the digits of
// its small entropy. With the row's own m, s and u: log sum = ln s, entropy = ln 2 (log2 s - u / s). An
// element of -inf gives s nothing, and u nothing because d is taken as -200 at the least; a NaN or +inf
// makes s a NaN, which is how a row that has no distribution is told.
//
// A row is read in slots of eight elements that start at 16-byte boundaries of memory, whatever the
// row's own alignment; the slots at its ends are read element by element. Rows are split over workgroups
// where there are few of them; the workgroup that finishes a row last (a ticket) joins its parts in their
// order. Nothing waits on another workgroup.
#include <algorithm>

#include "head_device.h"

namespace lg {
namespace {

using namespace head_detail;

constexpr int UNROLL = 4;  // slots a thread loads before it uses the first
constexpr uint32_t TICKETS = SK_COUNTER_BYTES / sizeof(uint32_t);
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.69314718055994530942;
constexpr float INF = __builtin_inff();
constexpr float FAR = -200.0f;  // below it 2^d is zero in f32

__device__ inline float exp2_fast(float d) { return __builtin_amdgcn_exp2f(d); }

// A row's m and, relative to it, s and u; or those of a part of it.
struct Part {
    float m;
    float pad;
    double s, u;
};

// What a pass leaves of a row for its gradient.
struct RowInfo {
    float m, log2s;
    float scale;  // the gradient is scale * p_j less the teacher's; 0: all zeros; NaN: all NaN
    float norm;   // log of the teacher's normalizer
};

struct PassArgs {
    const char* x;
    int64_t x_pitch;
    uint32_t row0, cols;
    uint32_t segs, seg_slots;  // workgroups to a row, slots to a workgroup
    float c, temperature;      // log2(e) / temperature
    Part* parts;               // [row - row0][segs]
    uint64_t* part_keys;       // [row - row0][segs][k]
    uint32_t* tickets;         // zero between launches
    LogprobArgs lp;
    DistillArgs ds;
    RowInfo* info;  // [row - row0], or null
};

// A row's slots.
template <uint32_t DT>
struct Slots {
    const char* base;  // of slot 0: the row's start rounded down to 16 bytes
    uint32_t head;     // elements of slot 0 before the row
    uint32_t cols, count;

    __device__ inline Slots(const char* row, uint32_t n) {
        head = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15) / elem_size<DT>;
        base = row - head * elem_size<DT>;
        cols = n;
        count = n == 0 ? 0 : (head + n + 7) / 8;
    }
    // Index in the row of slot j's first element, negative for one before it.
    __device__ inline int32_t first(uint32_t j) const { return static_cast<int32_t>(j * 8 - head); }
    // All eight inside the row: from the first such slot on, (head + cols) / 8 in all.
    __device__ inline bool whole(uint32_t j) const { return j - (head != 0) < (head + cols) / 8 - (head != 0); }
    __device__ inline bool has(uint32_t j, uint32_t e) const { return j * 8 + e - head < cols; }
    // Slot j; what lies outside the row is -inf.
    __device__ inline void load(uint32_t j, Run<DT>& r) const {
        if (whole(j)) {
            r.load(base + static_cast<uint64_t>(j) * 8 * elem_size<DT>);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const char* p = base + (static_cast<uint64_t>(j) * 8 + e) * elem_size<DT>;
            const bool inside = has(j, e);
            if constexpr (DT == LG_DTYPE_F32) {
                r.w[e / 4][e % 4] = inside ? *reinterpret_cast<const uint32_t*>(p) : 0xff800000u;
            } else {
                const uint32_t none = DT == LG_DTYPE_BF16 ? 0xff80u : 0xfc00u;
                const uint32_t bits = inside ? *reinterpret_cast<const uint16_t*>(p) : none;
                r.w[0][e / 2] = e % 2 ? (r.w[0][e / 2] & 0xffffu) | bits << 16 : bits;
            }
        }
    }
};

// A slot's maximum in LDS: its own 16 bits, or f32.
template <uint32_t DT>
struct SlotMax {
    typedef uint16_t T;
    static __device__ inline T pack(float v) {
        if constexpr (DT == LG_DTYPE_BF16) {
            return static_cast<uint16_t>(__float_as_uint(v) >> 16);
        } else {
            return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
        }
    }
    static __device__ inline float unpack(T b) { return widen<DT>(b); }
};
template <>
struct SlotMax<LG_DTYPE_F32> {
    typedef float T;
    static __device__ inline T pack(float v) { return v; }
    static __device__ inline float unpack(T b) { return b; }
};

// f32 as whole numbers of the same order; -0 counts as +0. No number gives 0.
__device__ inline uint32_t order(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ inline float unorder(uint32_t o) { return __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o); }
// Larger for a larger logit, and for a lower index among equal ones.
__device__ inline uint64_t key_of(float v, uint32_t index) { return static_cast<uint64_t>(order(v)) << 32 | (0xffffffffu - index); }
__device__ inline float key_value(uint64_t k) { return unorder(static_cast<uint32_t>(k >> 32)); }
__device__ inline uint32_t key_index(uint64_t k) { return 0xffffffffu - static_cast<uint32_t>(k); }

typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

// What a workgroup of T threads, T / 64 waves, keeps in LDS.
template <int T>
struct Shared {
    static constexpr int WAVES = T / 64;
    static constexpr uint32_t SLOT_BYTES = T == 64 ? 4096 : 16384;  // of the slots' maxima: 2 or 4 bytes each
    static constexpr uint32_t KEYS = SLOT_BYTES / 8;                // which take the maxima's place
    static constexpr uint32_t LIST = T == 64 ? 64 : 512;            // slots whose elements are looked at
    static constexpr uint32_t COUNTS = 96;                          // three for each two bits of a key
    alignas(16) uint64_t wide[KEYS];
    uint64_t best[TOP_MAX];
    float tops[T];
    uint32_t list[LIST];
    double s[WAVES], u[WAVES];
    float m[WAVES];
    float bound;  // below the k-th largest
    uint32_t listed, found, counts[COUNTS];
    bool last;
};

// The largest number that at least k of `tops`' T values reach, to sixteen bits of its order and from below; -inf
// where fewer than k are above -inf. FOLD: that many of the largest of each lane's values do. Two bits a step, by one wave.
template <int T, bool FOLD>
__device__ inline float threshold(const float* tops, uint32_t k) {
    constexpr int N = FOLD ? 1 : T / 64;
    const uint32_t lane = threadIdx.x % 64;
    float v[T / 64];
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v[i] = tops[i * 64 + lane];
    if (FOLD) {
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v[0] = fmaxf(v[0], v[i]);
    }
    uint32_t o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = order(v[i]) >> 16;
    uint32_t t = 0;
#pragma unroll
    for (int shift = 14; shift >= 0; shift -= 2) {
        uint32_t n[3] = {0, 0, 0};
#pragma unroll
        for (uint32_t c = 0; c < 3; ++c) {
#pragma unroll
            for (int i = 0; i < N; ++i) n[c] += __popcll(__ballot(o[i] >= (t | (c + 1) << shift)));
        }
        t |= (n[2] >= k ? 3u : n[1] >= k ? 2u : n[0] >= k ? 1u : 0u) << shift;
    }
    return t <= 0x007fu ? -INF : unorder(t << 16);
}

// How many of the workgroup's threads' `mine` there are in all.
template <int T>
__device__ inline uint32_t total(Shared<T>& sh, uint32_t mine) {
    __syncthreads();
    if (threadIdx.x == 0) sh.counts[0] = 0;
    __syncthreads();
    mine = wave_sum(mine);
    if (threadIdx.x % 64 == 0) atomicAdd(&sh.counts[0], mine);
    __syncthreads();
    return sh.counts[0];
}

// The largest number that at least k of n keys reach, told from bit `bits` - 1 down to bit `end`, two bits at a time (both
// even); `t` has the bits above. With k keys that differ from one another and all bits, the k-th largest key.
template <int T, typename F>
__device__ uint64_t kth_key(Shared<T>& sh, uint64_t t, uint32_t bits, uint32_t end, uint32_t n, uint32_t k, F&& key) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < Shared<T>::COUNTS; i += T) sh.counts[i] = 0;
    __syncthreads();
    uint32_t* count = sh.counts;
    for (uint32_t shift = bits; shift != end; count += 3) {
        shift -= 2;
        uint32_t c[3] = {0, 0, 0};
        for (uint32_t i = threadIdx.x; i < n; i += T) {
            const uint64_t v = key(i);
#pragma unroll
            for (uint64_t q = 0; q < 3; ++q) c[q] += v >= (t | (q + 1) << shift) ? 1 : 0;
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            c[q] = wave_sum(c[q]);
            if (threadIdx.x % 64 == 0) atomicAdd(&count[q], c[q]);
        }
        __syncthreads();
        t |= (count[2] >= k ? 3ull : count[1] >= k ? 2ull : count[0] >= k ? 1ull : 0ull) << shift;
    }
    return t;
}

// Keeps of the n keys in sh.wide those that can be among the k largest, told by the first sixteen bits, or where equal
// ones are too many by all; returns how many.
template <int T>
__device__ uint32_t narrow(Shared<T>& sh, uint32_t n, uint32_t k) {
    constexpr uint32_t HELD = Shared<T>::KEYS / T;
    uint64_t held[HELD];
#pragma unroll
    for (uint32_t i = 0; i < HELD; ++i) held[i] = i * T + threadIdx.x < n ? sh.wide[i * T + threadIdx.x] : 0;
    auto keep = [&](uint64_t bound) {
        __syncthreads();
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i) {
            if (held[i] != 0 && held[i] >= bound) sh.wide[atomicAdd(&sh.found, 1u)] = held[i];
        }
        __syncthreads();
        return sh.found;
    };
    auto key = [&](uint32_t i) { return sh.wide[i]; };
    const uint64_t t = kth_key(sh, 0, 64, 48, n, k, key);
    n = keep(t);
    return n <= 2 * T ? n : keep(kth_key(sh, t, 48, 0, n, k, key));
}

// sh.best, zeros so far, = the k largest of the n keys in sh.wide, in order: each key goes to the place that as
// many others exceed it, counted by two lanes, eight pairs each at a time (60 rows of 1505, 64
// alternatives: 7.3 us, by one lane 7.6, by four 7.6, by eight 7.8). Keys differ from one another.
template <int T>
__device__ inline void rank_keys(Shared<T>& sh, uint32_t n, uint32_t k) {
    constexpr uint32_t LANES = 2, PAIRS = 8;
    if (n > 2 * T) n = narrow(sh, n, k);  // a row of 1000 with 128 alternatives, all of them keys, 13 us; by ranks alone 48
    const uint32_t part = threadIdx.x % LANES, end = (n + 2 * LANES * PAIRS - 1) / (2 * LANES * PAIRS) * (2 * LANES * PAIRS);
    if (n + threadIdx.x < end) sh.wide[n + threadIdx.x] = 0;
    __syncthreads();
    const u64x2* pairs = reinterpret_cast<const u64x2*>(sh.wide);
    for (uint32_t i = threadIdx.x / LANES; i < n; i += T / LANES) {
        const uint64_t mine = sh.wide[i];
        uint32_t above = 0;
        for (uint32_t j = part; j < end / 2; j += LANES * PAIRS) {
            u64x2 v[PAIRS];
#pragma unroll
            for (uint32_t q = 0; q < PAIRS; ++q) v[q] = pairs[j + q * LANES];
#pragma unroll
            for (uint32_t q = 0; q < PAIRS; ++q) above += (v[q][0] > mine ? 1 : 0) + (v[q][1] > mine ? 1 : 0);
        }
#pragma unroll
        for (uint32_t d = 1; d < LANES; d *= 2) above += __shfl_xor(above, d);
        if (part == 0 && above < k) sh.best[above] = mine;
    }
    __syncthreads();
}

// sh.best = the k largest keys of slots [lo, hi), whose maxima are in sh.wide and whose threads' maxima
// are `mine`. An alternative lies in a slot whose maximum is one of the k largest, so slots below sh.bound, at
// most the k-th largest of the threads' maxima, drop out. Should too much remain (many equal logits, or a few threads
// with all of the largest), the k largest slots themselves are found, the lower of equal ones first. sh.listed and
// sh.found are zero, sh.best zeros.
template <uint32_t DT, int T>
__device__ void top_of_slots(Shared<T>& sh, const Slots<DT>& row, uint32_t lo, uint32_t hi, float mine, uint32_t k) {
    typedef SlotMax<DT> Max;
    const typename Max::T* maxima = reinterpret_cast<const typename Max::T*>(sh.wide);
    const uint32_t tid = threadIdx.x, n = hi - lo;
    float t = sh.bound;
    if (mine >= t) {
#pragma unroll 4
        for (uint32_t i = tid; i < n; i += T) {
            const float v = Max::unpack(maxima[i]);
            if (v >= t && v > -INF) {
                const uint32_t at = atomicAdd(&sh.listed, 1u);
                if (at < Shared<T>::LIST) sh.list[at] = i;
            }
        }
    }
    __syncthreads();
    uint32_t listed = sh.listed;
    // Element i % 8 of the list's slot i / 8, -inf for one outside the row.
    auto element = [&](uint32_t i, uint32_t* index) {
        const uint32_t j = lo + sh.list[i / 8];
        *index = row.first(j) + i % 8;
        return row.has(j, i % 8) ? load_one<DT>(row.base + (static_cast<uint64_t>(j) * 8 + i % 8) * elem_size<DT>) : -INF;
    };
    bool many = listed > Shared<T>::LIST;
    if (!many && listed * 8 > Shared<T>::KEYS) {
        uint32_t c = 0, index;
        for (uint32_t i = tid; i < listed * 8; i += T) c += element(i, &index) >= t ? 1 : 0;
        many = total(sh, c) > Shared<T>::KEYS;
    }
    if (many) {
        // A slot's maximum, without the bits that its type leaves zero, above the slot's number.
        constexpr uint32_t DROPPED = DT == LG_DTYPE_F32 ? 0 : DT == LG_DTYPE_BF16 ? 16 : 12, NUMBER = 14;
        static_assert(Shared<T>::SLOT_BYTES / elem_size<DT> <= 1u << NUMBER, "slots have their numbers");
        auto slot = [&](uint32_t i) {
            return static_cast<uint64_t>(order(Max::unpack(maxima[i])) >> DROPPED) << NUMBER | ((1u << NUMBER) - 1 - i);
        };
        const uint64_t bound = kth_key(sh, 0, 32 - DROPPED + NUMBER, 0, n, k, slot);
        t = unorder(static_cast<uint32_t>(bound >> NUMBER) << DROPPED);
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += T) {
            if (slot(i) >= bound) sh.list[atomicAdd(&sh.listed, 1u)] = i;
        }
        __syncthreads();
        listed = sh.listed;  // k
    }
    for (uint32_t i = tid; i < listed * 8; i += T) {
        uint32_t index;
        const float v = element(i, &index);
        if (v >= t && v > -INF) sh.wide[atomicAdd(&sh.found, 1u)] = key_of(v, index);
    }
    __syncthreads();
    rank_keys(sh, sh.found, k);
}

// The joined sums of the workgroup's threads, each relative to its own m; and for `k` > 0 in sh.bound at most the
// k-th largest of the threads' values `mine`, which the first wave finds while the others add.
template <bool ENTROPY, int T>
__device__ inline Part join(Shared<T>& sh, float m, double s, double u, float c, uint32_t k, float mine) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    float top = wave_max(m);
    if (lane == 0) sh.m[wave] = top;
    if (k > 0) sh.tops[threadIdx.x] = mine;
    __syncthreads();
    if (k > 0 && wave == 0) {
        // For few alternatives the maxima of groups of threads bound the k-th largest closely enough.
        const float t = k <= 24 ? threshold<T, true>(sh.tops, k) : threshold<T, false>(sh.tops, k);
        if (lane == 0) sh.bound = t;
    }
#pragma unroll
    for (int w = 0; w < Shared<T>::WAVES; ++w) top = fmaxf(top, sh.m[w]);
    if (m != -INF) {  // else s and u are zero, or NaN
        const float shift = (m - top) * c;
        const double f = exp2_fast(shift);
        if (ENTROPY) u = f * (u + fmaxf(shift, 4 * FAR) * s);
        s = f * s;
    }
    s = wave_sum(s);
    if (ENTROPY) u = wave_sum(u);
    if (lane == 0) {
        sh.s[wave] = s;
        if (ENTROPY) sh.u[wave] = u;
    }
    __syncthreads();
    Part p{top, 0.0f, 0.0, 0.0};
#pragma unroll
    for (int w = 0; w < Shared<T>::WAVES; ++w) {
        p.s += sh.s[w];
        if (ENTROPY) p.u += sh.u[w];
    }
    return p;
}

// Writes what is asked of a row with sums p and, for k > 0, its best keys in sh.best.
template <int T>
__device__ inline void finish_logprobs(const PassArgs& a, const Shared<T>& sh, bool named, float logit, uint32_t row, Part p) {
    const LogprobArgs& o = a.lp;
    const uint32_t tid = threadIdx.x;
    const bool bad = p.s != p.s, empty = !bad && p.m == -INF;
    const double log_s = empty ? 0.0 : log(p.s);
    const float nan = __builtin_nanf("");
    if (tid == 0) {
        if (o.tokens != nullptr) {
            float v = 0.0f;
            if (named) v = bad ? nan : static_cast<float>(static_cast<double>(logit - (empty ? 0.0f : p.m)) / o.temperature - log_s);
            o.logprobs[row] = v;
        }
        if (o.entropy != nullptr) o.entropy[row] = bad ? nan : empty ? 0.0f : static_cast<float>(log_s - LN2 * (p.u / p.s));
        if (o.stats != nullptr) {
            o.stats[row * o.stats_pitch] = bad ? nan : p.m;
            o.stats[row * o.stats_pitch + 1] = bad ? nan : empty ? -INF : static_cast<float>(log_s);
        }
    }
    for (uint32_t i = tid; i < o.k; i += T) {
        const uint64_t key = bad ? 0 : sh.best[i];
        o.top_ids[row * o.ids_pitch + i] = key == 0 ? -1 : static_cast<int32_t>(key_index(key));
        const float v = key == 0 ? -INF : static_cast<float>(static_cast<double>(key_value(key) - p.m) / o.temperature - log_s);
        o.top[row * o.top_pitch + i] = bad ? nan : v;
    }
}

// Whether entry i of a row's list names one of `cols` logits with a probability, and its log.
struct Teacher {
    const int32_t* ids;
    const float* values;
    uint32_t k, cols;
    __device__ inline Teacher(const DistillArgs& a, uint32_t row) {
        ids = a.ids + row * a.ids_pitch;
        values = a.values + row * a.values_pitch;
        k = a.k;
        cols = a.cols;
    }
    __device__ inline bool named(uint32_t i, uint32_t* id, float* value) const {
        if (i >= k || ids[i] < 0 || static_cast<uint32_t>(ids[i]) >= cols || values[i] == -INF) return false;
        *id = static_cast<uint32_t>(ids[i]);
        *value = values[i];
        return true;
    }
};

// The teacher's list of a row in one wave: each lane holds two of its entries.
struct Entries {
    uint32_t id[2];
    float value[2], logit[2];
    bool named[2], any;
    double norm;  // log of the normalizer

    // `logits`: reads the student's logits at the entries, too.
    template <uint32_t DT>
    __device__ inline void load(const DistillArgs& o, const char* x, uint32_t row) {
        const uint32_t lane = threadIdx.x % 64;
        const Teacher teacher(o, row);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            value[i] = -INF;
            id[i] = 0;
            named[i] = teacher.named(lane + 64 * i, &id[i], &value[i]);
            logit[i] = named[i] ? load_one<DT>(x + static_cast<uint64_t>(id[i]) * elem_size<DT>) : 0.0f;
        }
    }
    __device__ inline void normalize(const DistillArgs& o) {
        any = __ballot(named[0] || named[1]) != 0;
        norm = 0.0;
        if (!o.normalize) return;
        float top = fmaxf(named[0] ? value[0] : -INF, named[1] ? value[1] : -INF);
        top = wave_max(top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (named[i]) sum += exp(static_cast<double>(value[i]) - top);
        }
        norm = top + log(wave_sum(sum));
    }
    // The mass sum p_i and, relative to the student's normalizer, the loss: sum p_i (log p_i - (x_i - m) / T).
    __device__ inline void sums(const DistillArgs& o, float m, double* mass, double* loss) const {
        *mass = *loss = 0.0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!named[i]) continue;
            const double lp = value[i] - norm, q = exp(lp);
            *mass += q;
            if (q != 0.0) *loss += q * (lp - static_cast<double>(logit[i] - m) / o.temperature);
        }
        *mass = wave_sum(*mass);
        *loss = wave_sum(*loss);
    }
};

// A row's loss and what its gradient needs, by one wave.
__device__ inline RowInfo finish_distill(const DistillArgs& o, const Entries& list, uint32_t row, Part p, double mass, double loss) {
    const bool bad = p.s != p.s, empty = !bad && p.m == -INF;
    const float weight = (o.weights != nullptr ? o.weights[row] : 1.0f) * o.temperature, nan = __builtin_nanf("");
    const bool idle = empty || weight == 0.0f || !list.any;
    const double log_s = empty ? 0.0 : log(p.s);
    if (threadIdx.x % 64 == 0) o.losses[row] = idle ? 0.0f : bad ? nan : static_cast<float>((loss + mass * log_s) * weight * o.temperature);
    return RowInfo{p.m, static_cast<float>(log_s / LN2), idle ? 0.0f : bad ? nan : static_cast<float>(mass * weight), static_cast<float>(list.norm)};
}

// This wave's device-scope stores have reached memory. They go past the L2 (each XCD has its own) and are
// read past it by device-scope loads, so a ticket drawn after this says that they are there; a release fence
// would write back the whole L2, which costs every workgroup 0.1 us in turn (the pass over 48 rows of 100003, 528
// workgroups: 42 us with it, 12 without).
__device__ inline void written() {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The joined parts of row `at`, by the workgroup that wrote the last of them; with TOP their best keys in sh.best.
template <bool ENTROPY, bool TOP, int T>
__device__ Part join_parts(const PassArgs& a, Shared<T>& sh, uint32_t at) {
    const uint32_t tid = threadIdx.x, k = TOP ? a.lp.k : 0, all = a.segs * k;
    if (tid == 0) __hip_atomic_store(a.tickets + at, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    auto key = [&](uint32_t i) {
        return __hip_atomic_load(a.part_keys + static_cast<uint64_t>(at) * all + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    // The threads' largest keys bound the k-th of all from below, closely where a thread's keys are of differing
    // ranks in the parts' sorted lists. Up to HELD keys a thread stay in registers.
    auto turn = [&](uint32_t i) { return i * T + (tid + 83 * i) % T; };
    constexpr int HELD = 8;
    uint64_t held[HELD];
    float mine = -INF;
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) held[i] = turn(i) < all ? key(turn(i)) : 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) mine = held[i] != 0 ? fmaxf(mine, key_value(held[i])) : mine;
        for (uint32_t i = HELD; i * T < all; ++i) {
            const uint64_t v = turn(i) < all ? key(turn(i)) : 0;
            if (v != 0) mine = fmaxf(mine, key_value(v));
        }
        for (uint32_t i = tid; i < TOP_MAX; i += T) sh.best[i] = 0;
        if (tid == 0) sh.found = 0;
    }
    // Each thread joins the parts of its turn, in order.
    float m = -INF;
    double s = 0.0, u = 0.0;
    for (uint32_t i = tid; i < a.segs; i += T) {
        const Part* q = a.parts + static_cast<uint64_t>(at) * a.segs + i;
        const float qm = __hip_atomic_load(&q->m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const double qs = __hip_atomic_load(&q->s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const double qu = ENTROPY ? __hip_atomic_load(&q->u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
        const float ref = fmaxf(m, qm);
        const float f = ref == -INF ? 0.0f : fmaxf((m - ref) * a.c, 4 * FAR), g = ref == -INF ? 0.0f : fmaxf((qm - ref) * a.c, 4 * FAR);
        u = exp2_fast(f) * (u + f * s) + exp2_fast(g) * (qu + g * qs);
        s = exp2_fast(f) * s + exp2_fast(g) * qs;
        m = ref;
    }
    const Part p = join<ENTROPY>(sh, m, s, u, a.c, k, mine);
    if constexpr (TOP) {
        const float t = sh.bound;
        auto push = [&](uint64_t v) {
            const uint32_t to = atomicAdd(&sh.found, 1u);
            if (to < Shared<T>::KEYS) sh.wide[to] = v;
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (held[i] != 0 && key_value(held[i]) >= t) push(held[i]);
        }
        for (uint32_t i = HELD * T + tid; i < all; i += T) {
            const uint64_t v = key(i);
            if (v != 0 && key_value(v) >= t) push(v);
        }
        __syncthreads();
        if (sh.found > Shared<T>::KEYS) {  // many equal ones
            const uint64_t bound = kth_key(sh, 0, 64, 0, all, k, key);
            if (tid == 0) sh.found = 0;
            __syncthreads();
            for (uint32_t i = tid; i < all; i += T) {
                const uint64_t v = key(i);
                if (v != 0 && v >= bound) push(v);
            }
            __syncthreads();
        }
        rank_keys(sh, sh.found, k);
    }
    return p;
}

// A workgroup's part of a row.
template <uint32_t DT>
struct Piece {
    uint32_t at, seg, row;  // at: row - row0
    const char* x;
    Slots<DT> slots;
    uint32_t lo, hi;  // slots of the part
    bool live;        // a row without weight is not read
    __device__ inline Piece(const PassArgs& a, uint32_t item)
        : at(item / a.segs), seg(item % a.segs), row(a.row0 + at), x(a.x + row * a.x_pitch * elem_size<DT>), slots(x, a.cols) {
        lo = min(seg * a.seg_slots, slots.count);
        hi = min(lo + a.seg_slots, slots.count);
        live = a.ds.weights == nullptr || a.ds.weights[row] != 0.0f;
    }
};

// A pass over a part of a row; the row's last workgroup finishes it. Bound by reading the logits, and by the latency of
// what follows a row's last slot, under which other rows' workgroups of the compute unit read: 4096 rows of 32768 bf16
// 44 us without entropy and alternatives (6.0 TB/s), 51 us with entropy, 58 and 64 us with 20 and 64 alternatives (by
// workgroups of eight waves 57, 67 and 73 us); one row of 131072 with 20 alternatives 10.1 us, 48 rows of 100003 f32 with a
// teacher 10 us.
template <uint32_t DT, bool ENTROPY, bool TOP, bool DISTILL, int T>
__global__ __launch_bounds__(T) void row_pass(PassArgs a) {
    __shared__ Shared<T> sh;
    const uint32_t tid = threadIdx.x;
    typename SlotMax<DT>::T* maxima = reinterpret_cast<typename SlotMax<DT>::T*>(sh.wide);
    const Piece<DT> now(a, blockIdx.x);
    if constexpr (DISTILL) {
        if (!now.live) {
            if (tid == 0 && now.seg == 0) {
                a.ds.losses[now.row] = 0.0f;
                if (a.info != nullptr) a.info[now.at] = RowInfo{0.0f, 0.0f, 0.0f, 0.0f};
            }
            return;
        }
    }
    // What the row's end needs beside its sums is asked for here, so that its latency passes under the row's own.
    Entries list;
    float logit = 0.0f;
    bool named = false;
    if constexpr (DISTILL) {
        if (tid < 64) list.load<DT>(a.ds, now.x, now.row);
    } else if (a.lp.tokens != nullptr) {
        const int32_t t = a.lp.tokens[now.row];
        named = t >= 0 && static_cast<uint32_t>(t) < a.cols;
        if (named) logit = load_one<DT>(now.x + static_cast<uint64_t>(t) * elem_size<DT>);
    }
    if constexpr (TOP) {
        for (uint32_t i = tid; i < TOP_MAX; i += T) sh.best[i] = 0;
        if (tid == 0) sh.listed = sh.found = 0;
    }
    float m = -INF;
    double s = 0.0, u = 0.0;
    for (uint32_t j0 = now.lo + tid; j0 < now.hi; j0 += T * UNROLL) {
        Run<DT> r[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const uint32_t j = j0 + i * T;
            if (j < now.hi) {
                now.slots.load(j, r[i]);
            } else {
                r[i].clear();
            }
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            float v = r[i][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) v = fmaxf(v, r[i][e]);
            if (TOP && j0 + i * T < now.hi) maxima[j0 + i * T - now.lo] = SlotMax<DT>::pack(v);
            top = fmaxf(top, v);
        }
        const float ref = top == -INF ? 0.0f : top, shift = fmaxf((m - ref) * a.c, 4 * FAR);
        const double f = exp2_fast(shift);
        if (ENTROPY) u = f * (u + shift * s);
        s = f * s;
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            float ps = 0.0f, pu = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = (r[i][e] - ref) * a.c, p = exp2_fast(d);
                ps += p;
                if (ENTROPY) pu = __builtin_fmaf(p, fmaxf(d, FAR), pu);
            }
            s += ps;
            if (ENTROPY) u += pu;
        }
        m = top;
    }
    Part p = join<ENTROPY>(sh, m, s, u, a.c, TOP ? a.lp.k : 0, m);
    if constexpr (TOP) top_of_slots<DT>(sh, now.slots, now.lo, now.hi, m, a.lp.k);
    if (a.segs > 1) {
        // Thread 0 writes the part and draws the ticket; the keys are wave 0's.
        if (tid < 64) {
            if constexpr (TOP) {
                uint64_t* keys = a.part_keys + (static_cast<uint64_t>(now.at) * a.segs + now.seg) * a.lp.k;
                for (uint32_t i = tid; i < a.lp.k; i += 64) __hip_atomic_store(keys + i, sh.best[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            if (tid == 0) {
                Part* to = a.parts + static_cast<uint64_t>(now.at) * a.segs + now.seg;
                __hip_atomic_store(&to->m, p.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(&to->s, p.s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (ENTROPY) __hip_atomic_store(&to->u, p.u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            written();
            if (tid == 0) sh.last = __hip_atomic_fetch_add(a.tickets + now.at, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.segs - 1;
        }
        __syncthreads();
        if (!sh.last) return;
        p = join_parts<ENTROPY, TOP>(a, sh, now.at);
    }
    if constexpr (DISTILL) {
        if (tid < 64) {
            list.normalize(a.ds);
            double mass, loss;
            list.sums(a.ds, p.m, &mass, &loss);
            const RowInfo info = finish_distill(a.ds, list, now.row, p, mass, loss);
            if (a.info != nullptr && tid == 0) a.info[now.at] = info;
        }
    } else {
        finish_logprobs(a, sh, named, logit, now.row, p);
    }
}

// ------------------------------------------------------------------------------- gradients

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_UNROLL = 4;
constexpr uint32_t GRAD_SLOTS = GRAD_THREADS * GRAD_UNROLL;  // of a workgroup

struct GradArgs {
    const char* x;
    char* dx;
    int64_t x_pitch, dx_pitch;
    uint32_t row0, cols, segs;
    float c, inverse;  // log2(e) / temperature, 1 / temperature
    LogprobBackArgs lp;
    DistillArgs ds;
    const RowInfo* info;
};

// What the teacher takes from logit `id`: an id that the list holds twice loses the sum of both, in the list's order.
// (One entry at a time its reads' latencies add up: 83 rows of 1731 with 128 entries 11.8 us, so 6.7.)
__device__ inline float taken(const uint32_t* ids, const float* minus, uint32_t k, uint32_t id) {
    float v = 0.0f;
    for (uint32_t i = 0; i < k; i += 16) {
        u32x4 n[4];
        f32x4 m[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            n[q] = reinterpret_cast<const u32x4*>(ids + i)[q];
            m[q] = reinterpret_cast<const f32x4*>(minus + i)[q];
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) v += n[q / 4][q % 4] == id ? m[q / 4][q % 4] : 0.0f;
    }
    return v;
}

enum GradMode { LOGPROB, LOGPROB_ENTROPY, TEACHER };

// dx of GRAD_SLOTS slots of a row: an element at a time from the row's statistics. The token's own term
// joins in its slot; a teacher's are written over the dense gradient when it is complete, from logits read before. Bound by
// memory: 1024 rows of 50001 f32 83.5 us (4.9 TB/s).
template <uint32_t DT, GradMode MODE>
__global__ __launch_bounds__(GRAD_THREADS) void grad_rows(GradArgs a) {
    const uint32_t tid = threadIdx.x, at = blockIdx.x / a.segs, seg = blockIdx.x % a.segs, row = a.row0 + at;
    const char* x = a.x + row * a.x_pitch * elem_size<DT>;
    char* dx = a.dx + row * a.dx_pitch * elem_size<DT>;
    const Slots<DT> slots(x, a.cols);
    float m, log2s, g = 0.0f, h = 0.0f, entropy = 0.0f, scale = 1.0f;
    int32_t token = -1;
    if constexpr (MODE == TEACHER) {
        const RowInfo info = a.info[at];
        m = info.m;
        log2s = info.log2s;
        scale = info.scale;
    } else {
        m = a.lp.stats[row * a.lp.stats_pitch];
        log2s = a.lp.stats[row * a.lp.stats_pitch + 1] * LOG2E;
        if (m == -INF) scale = 0.0f;
        token = a.lp.tokens[row];
        if (token >= static_cast<int32_t>(a.cols)) token = -1;
        if (token >= 0) g = a.lp.dlogprobs[row] * a.inverse;
        if constexpr (MODE == LOGPROB_ENTROPY) {
            h = a.lp.dentropy[row] * a.inverse;
            entropy = a.lp.entropy[row];
        }
    }
    // One slot's gradient, from its logits.
    auto gradient = [&](const Run<DT>& r, int32_t first, float (&o)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = (r[e] - m) * a.c - log2s, p = exp2_fast(d);
            if constexpr (MODE == TEACHER) {
                o[e] = scale * p;
            } else if constexpr (MODE == LOGPROB) {
                o[e] = -g * p;
            } else {
                o[e] = -p * __builtin_fmaf(h, __builtin_fmaf(fmaxf(d, FAR), static_cast<float>(LN2), entropy), g);
            }
            if constexpr (MODE != TEACHER) {
                if (first + e == token) o[e] += g;
            }
        }
    };
    __shared__ __attribute__((aligned(16))) uint32_t ids[TOP_MAX];
    __shared__ __attribute__((aligned(16))) float minus[TOP_MAX];
    __shared__ float own[TOP_MAX];
    const uint32_t lo = seg * GRAD_SLOTS;
    if constexpr (MODE == TEACHER) {
        // The list's entries that lie in these slots: their probabilities, and their logits' own before any is overwritten.
        if (tid < TOP_MAX) {
            uint32_t id = 0xffffffffu;
            float value = 0.0f;
            const Teacher teacher(a.ds, row);
            ids[tid] = 0xffffffffu;
            if (scale != 0.0f && teacher.named(tid, &id, &value)) {
                const float weight = (a.ds.weights != nullptr ? a.ds.weights[row] : 1.0f) * a.ds.temperature;
                minus[tid] = weight * exp2_fast((value - a.info[at].norm) * LOG2E);
                ids[tid] = id;
                const uint32_t j = (id + slots.head) / 8;
                if (j >= lo && j < lo + GRAD_SLOTS) {
                    own[tid] = scale * exp2_fast((load_one<DT>(x + static_cast<uint64_t>(id) * elem_size<DT>) - m) * a.c - log2s);
                }
            }
        }
        __syncthreads();
    }
    Run<DT> r[GRAD_UNROLL];
#pragma unroll
    for (int i = 0; i < GRAD_UNROLL; ++i) {
        const uint32_t j = lo + i * GRAD_THREADS + tid;
        if (j < slots.count && scale != 0.0f) slots.load(j, r[i]);
    }
#pragma unroll
    for (int i = 0; i < GRAD_UNROLL; ++i) {
        const uint32_t j = lo + i * GRAD_THREADS + tid;
        if (j >= slots.count) break;
        float o[8] = {};
        if (scale != 0.0f) gradient(r[i], slots.first(j), o);
        if (slots.whole(j)) {
            store_run<DT>(dx + slots.first(j) * static_cast<int64_t>(elem_size<DT>), o);
        } else {
            for (int e = 0; e < 8; ++e) {
                if (slots.has(j, e)) store_one<DT>(dx + (slots.first(j) + e) * static_cast<int64_t>(elem_size<DT>), o[e]);
            }
        }
    }
    if constexpr (MODE == TEACHER) {
        if (scale == 0.0f) return;
        __syncthreads();
        if (tid < TOP_MAX && ids[tid] != 0xffffffffu) {
            const uint32_t id = ids[tid], j = (id + slots.head) / 8;
            if (j >= lo && j < lo + GRAD_SLOTS) {
                store_one<DT>(dx + static_cast<uint64_t>(id) * elem_size<DT>, own[tid] - taken(ids, minus, a.ds.k, id));
            }
        }
    }
}

// Loss and gradient of whole rows, a workgroup each: the row stays in registers, NV slots a thread, from its one read
// to its gradient's one write. The first wave works out the teacher's list beside the sums. Bound by memory where
// at least two rows share a compute unit: 4096 rows of 65536 bf16 210 us (5.1 TB/s read and written, a large copy's rate), in
// two passes 306 us, with eight slots a thread and one row a compute unit 304 us.
template <uint32_t DT, int T, int NV>
__global__ __launch_bounds__(T) void distill_rows(GradArgs a) {
    constexpr int WAVES = T / 64;
    __shared__ double sums[WAVES];
    __shared__ float tops[WAVES];
    __shared__ __attribute__((aligned(16))) uint32_t ids[TOP_MAX];
    __shared__ __attribute__((aligned(16))) float minus[TOP_MAX];
    __shared__ float own[TOP_MAX];
    __shared__ RowInfo shared_info;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64, row = a.row0 + blockIdx.x;
    const char* x = a.x + row * a.x_pitch * elem_size<DT>;
    char* dx = a.dx + row * a.dx_pitch * elem_size<DT>;
    const Slots<DT> slots(x, a.cols);
    const float weight = a.ds.weights != nullptr ? a.ds.weights[row] : 1.0f;
    Run<DT> r[NV];
    RowInfo info{0.0f, 0.0f, 0.0f, 0.0f};
    if (weight != 0.0f) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t j = i * T + tid;
            if (j < slots.count) {
                slots.load(j, r[i]);
            } else {
                r[i].clear();
            }
        }
        Entries list;
        if (wave == 0) list.load<DT>(a.ds, x, row);
        float top = -INF;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, r[i][e]);
        }
        top = wave_max(top);
        if (lane == 0) tops[wave] = top;
        if (wave == 0) list.normalize(a.ds);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
        const float ref = top == -INF ? 0.0f : top;
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            r[i].keep();
            float ps = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ps += exp2_fast((r[i][e] - ref) * a.c);
            s += ps;
        }
        s = wave_sum(s);
        if (lane == 0) sums[wave] = s;
        double mass = 0.0, loss = 0.0;
        if (wave == 0) list.sums(a.ds, top, &mass, &loss);
        __syncthreads();
        if (wave == 0) {
            Part p{top, 0.0f, 0.0, 0.0};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) p.s += sums[w];
            info = finish_distill(a.ds, list, row, p, mass, loss);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ids[lane + 64 * i] = list.named[i] ? list.id[i] : 0xffffffffu;
                minus[lane + 64 * i] = weight * a.ds.temperature * exp2_fast((list.value[i] - info.norm) * LOG2E);
                own[lane + 64 * i] = info.scale * exp2_fast(__builtin_fmaf(list.logit[i] - info.m, a.c, -info.log2s));
            }
            if (lane == 0) shared_info = info;
        }
        __syncthreads();
        info = shared_info;
    } else if (tid == 0) {
        a.ds.losses[row] = 0.0f;
    }
    auto store = [&](uint32_t j, const float (&o)[8]) {
        if (slots.whole(j)) {
            store_run<DT>(dx + slots.first(j) * static_cast<int64_t>(elem_size<DT>), o);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (slots.has(j, e)) store_one<DT>(dx + (slots.first(j) + e) * static_cast<int64_t>(elem_size<DT>), o[e]);
            }
        }
    };
    if (info.scale == 0.0f) {
        const float zeros[8] = {};
        for (uint32_t j = tid; j < slots.count; j += T) store(j, zeros);
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t j = i * T + tid;
        if (j >= slots.count) break;
        r[i].keep();
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = info.scale * exp2_fast(__builtin_fmaf(r[i][e] - info.m, a.c, -info.log2s));
        store(j, o);
    }
    __syncthreads();
    if (tid < TOP_MAX && ids[tid] != 0xffffffffu) store_one<DT>(dx + static_cast<uint64_t>(ids[tid]) * elem_size<DT>, own[tid] - taken(ids, minus, a.ds.k, ids[tid]));
}

// ------------------------------------------------------------------------------- launches

uint32_t ceil_div(uint64_t a, uint64_t b) { return static_cast<uint32_t>((a + b - 1) / b); }

// Parts of a row, and slots to a part. Few rows are split until the chip has a workgroup for each compute unit, or two
// while a part has over 64 KB, and each thread four slots; more only cost tickets (16 rows of 131072 in 256 parts 13.9 us, in
// 512 15.9; 128 rows in 256 20.4, in 512 17.8). Rows that one workgroup reads in the time of a ticket and a join stay whole:
// up to 2048 slots (20 rows of 16000 with 20 alternatives 7.8 us, in parts 10.3), more with more rows (150 of 32000: 10.5 us,
// in two parts 13.3; 200 of 48000: 13.2 and 15.1). Where alternatives are wanted, no more slots than their maxima
// have room for in LDS.
struct Split {
    uint32_t segs, seg_slots;
};
constexpr int THREADS = 256;
Split split_rows(uint32_t rows, uint32_t cols, uint32_t size, uint32_t k) {
    const uint32_t slots = ceil_div(static_cast<uint64_t>(cols) + 7, 8) + 1, most = Shared<THREADS>::SLOT_BYTES / size;
    const uint32_t runs = static_cast<uint32_t>(static_cast<uint64_t>(cols) * size >> 16);
    uint32_t segs = std::max(ceil_div(256, rows), std::min(ceil_div(512, rows), runs));
    segs = slots <= (rows >= 128 ? 8192 : rows >= 16 ? 4096 : 2048) ? 1 : std::min(segs, ceil_div(slots, 4 * THREADS));
    if (k > 0) segs = std::max(std::min(segs, Shared<THREADS>::KEYS / k), ceil_div(slots, most));
    const uint32_t each = ceil_div(slots, segs);
    return {ceil_div(slots, each), each};
}

template <uint32_t DT, bool ENTROPY, bool TOP, bool DISTILL>
void launch_pass(lg_ctx* ctx, hipStream_t s, const PassArgs& a, uint32_t rows) {
    const uint32_t items = rows * a.segs;
    // Many short rows: a wave each, whose 64 maxima bound few alternatives closely enough (4096 rows of 4096 with 5
    // alternatives: 12.4 us, by workgroups of four waves 22 us).
    if (a.segs == 1 && rows >= 1024 && a.seg_slots <= Shared<64>::SLOT_BYTES / elem_size<DT> && a.seg_slots <= 1025 && a.lp.k <= 24) {
        hipLaunchKernelGGL((row_pass<DT, ENTROPY, TOP, DISTILL, 64>), dim3(items), dim3(64), 0, s, a);
    } else {
        hipLaunchKernelGGL((row_pass<DT, ENTROPY, TOP, DISTILL, THREADS>), dim3(items), dim3(THREADS), 0, s, a);
    }
    launched(ctx, DISTILL ? "row_pass_distill" : TOP ? "row_pass_top" : "row_pass");
}

// Rows in batches of `most`, and of no more than a launch's threads have 32-bit numbers for; the longest rows' parts are
// 2^18 workgroups, and fill 17 MB of scratch with their alternatives.
template <typename F>
void batches(uint32_t rows, uint64_t wgs_per_row, uint64_t most, F&& launch) {
    const uint64_t batch = std::min<uint64_t>(most, (1ull << 22) / wgs_per_row);
    for (uint64_t r = 0; r < rows; r += batch) launch(static_cast<uint32_t>(r), static_cast<uint32_t>(std::min<uint64_t>(batch, rows - r)));
}

// Rows whose parts fit the scratch and whose tickets there are.
uint64_t split_most(uint32_t segs, uint64_t bytes_per_row) {
    return std::min<uint64_t>(SPLIT_PARTIAL_MAX / bytes_per_row, segs > 1 ? TICKETS : UINT32_MAX);
}

template <uint32_t DT>
void logprobs_of(lg_ctx* ctx, hipStream_t s, const LogprobArgs& o) {
    const Split split = split_rows(o.rows, o.cols, elem_size<DT>, o.k);
    PassArgs a{};
    a.x = static_cast<const char*>(o.x);
    a.x_pitch = o.x_pitch;
    a.cols = o.cols;
    a.segs = split.segs;
    a.seg_slots = split.seg_slots;
    a.c = LOG2E / o.temperature;
    a.temperature = o.temperature;
    a.lp = o;
    const auto run = [&](void* scratch) {
        const uint64_t per_row = split.segs * (sizeof(Part) + o.k * sizeof(uint64_t));
        batches(o.rows, split.segs, split.segs == 1 ? o.rows : split_most(split.segs, per_row), [&](uint32_t r, uint32_t n) {
            a.row0 = r;
            if (scratch != nullptr) {
                a.tickets = reinterpret_cast<uint32_t*>(static_cast<char*>(scratch) + SPLIT_PARTIAL_MAX);
                a.parts = static_cast<Part*>(scratch);
                a.part_keys = reinterpret_cast<uint64_t*>(a.parts + static_cast<uint64_t>(n) * split.segs);
            }
            if (o.k > 0) {
                o.entropy != nullptr ? launch_pass<DT, true, true, false>(ctx, s, a, n) : launch_pass<DT, false, true, false>(ctx, s, a, n);
            } else {
                o.entropy != nullptr ? launch_pass<DT, true, false, false>(ctx, s, a, n) : launch_pass<DT, false, false, false>(ctx, s, a, n);
            }
        });
    };
    if (split.segs == 1) {
        run(nullptr);
    } else {
        with_split_scratch(ctx, s, run);
    }
}

template <uint32_t DT, GradMode MODE>
void launch_grad(lg_ctx* ctx, hipStream_t s, const GradArgs& a, uint32_t rows) {
    hipLaunchKernelGGL((grad_rows<DT, MODE>), dim3(rows * a.segs), dim3(GRAD_THREADS), 0, s, a);
    launched(ctx, MODE == TEACHER ? "grad_rows_distill" : "grad_rows");
}

uint32_t grad_segs(uint32_t cols) { return ceil_div((static_cast<uint64_t>(cols) + 7 + 7) / 8, GRAD_SLOTS); }

template <uint32_t DT>
void back_of(lg_ctx* ctx, hipStream_t s, const LogprobBackArgs& o) {
    GradArgs a{};
    a.x = static_cast<const char*>(o.x);
    a.dx = static_cast<char*>(o.dx);
    a.x_pitch = o.x_pitch;
    a.dx_pitch = o.dx_pitch;
    a.cols = o.cols;
    a.segs = grad_segs(o.cols);
    a.c = LOG2E / o.temperature;
    a.inverse = 1.0f / o.temperature;
    a.lp = o;
    batches(o.rows, a.segs, o.rows, [&](uint32_t r, uint32_t n) {
        a.row0 = r;
        o.dentropy != nullptr ? launch_grad<DT, LOGPROB_ENTROPY>(ctx, s, a, n) : launch_grad<DT, LOGPROB>(ctx, s, a, n);
    });
}

template <uint32_t DT, int T, int NV>
void launch_rows(lg_ctx* ctx, hipStream_t s, const GradArgs& a, uint32_t rows) {
    hipLaunchKernelGGL((distill_rows<DT, T, NV>), dim3(rows), dim3(T), 0, s, a);
    launched(ctx, "distill_rows");
}

// Whether whole rows fit a workgroup's registers (65536 f32 or 131072 16-bit logits); launches them if so. Rows past
// 65536 logits are split instead where they are too few to fill the chip (64 rows of 131072: 22 us against 24; of
// 65536 whole 14 us against 18).
template <uint32_t DT>
bool distill_whole_rows(lg_ctx* ctx, hipStream_t s, GradArgs a, uint32_t rows) {
    const bool aligned = (reinterpret_cast<uintptr_t>(a.x) | static_cast<uint64_t>(a.x_pitch * elem_size<DT>)) % 16 == 0;
    const uint64_t slots = (static_cast<uint64_t>(a.cols) + (aligned ? 0 : 16 / elem_size<DT> - 1) + 7) / 8;
    if (slots > (DT == LG_DTYPE_F32 ? 8 : 16) * 1024 || (slots > 8 * 1024 && rows < 96)) return false;
    batches(rows, 1, rows, [&](uint32_t r, uint32_t n) {
        a.row0 = r;
        if (slots <= 4 * 128) {
            launch_rows<DT, 128, 4>(ctx, s, a, n);
        } else if (slots <= 4 * 256) {
            launch_rows<DT, 256, 4>(ctx, s, a, n);
        } else if (slots <= 4 * 512) {
            launch_rows<DT, 512, 4>(ctx, s, a, n);
        } else if (slots <= 8 * 512) {
            launch_rows<DT, 512, 8>(ctx, s, a, n);
        } else if constexpr (DT == LG_DTYPE_F32) {
            launch_rows<DT, 1024, 8>(ctx, s, a, n);
        } else if (slots <= 16 * 512) {
            launch_rows<DT, 512, 16>(ctx, s, a, n);
        } else {
            launch_rows<DT, 1024, 16>(ctx, s, a, n);
        }
    });
    return true;
}

template <uint32_t DT>
void distill_of(lg_ctx* ctx, hipStream_t s, const DistillArgs& o) {
    const Split split = split_rows(o.rows, o.cols, elem_size<DT>, 0);
    PassArgs a{};
    a.x = static_cast<const char*>(o.x);
    a.x_pitch = o.x_pitch;
    a.cols = o.cols;
    a.segs = split.segs;
    a.seg_slots = split.seg_slots;
    a.c = LOG2E / o.temperature;
    a.temperature = o.temperature;
    a.ds = o;
    GradArgs g{};
    g.x = a.x;
    g.dx = static_cast<char*>(o.dx);
    g.x_pitch = o.x_pitch;
    g.dx_pitch = o.dx_pitch;
    g.cols = o.cols;
    g.segs = grad_segs(o.cols);
    g.c = a.c;
    g.ds = o;
    if (o.dx != nullptr && distill_whole_rows<DT>(ctx, s, g, o.rows)) return;
    with_split_scratch(ctx, s, [&](void* scratch) {
        const uint64_t per_row = sizeof(RowInfo) + (split.segs == 1 ? 0 : split.segs * sizeof(Part));
        batches(o.rows, std::max(split.segs, g.segs), split_most(split.segs, per_row), [&](uint32_t r, uint32_t n) {
            a.row0 = g.row0 = r;
            a.tickets = reinterpret_cast<uint32_t*>(static_cast<char*>(scratch) + SPLIT_PARTIAL_MAX);
            a.parts = static_cast<Part*>(scratch);
            RowInfo* info = reinterpret_cast<RowInfo*>(a.parts + (split.segs == 1 ? 0 : static_cast<uint64_t>(n) * split.segs));
            a.info = o.dx != nullptr ? info : nullptr;
            g.info = info;
            launch_pass<DT, false, false, true>(ctx, s, a, n);
            if (o.dx != nullptr && o.cols > 0) launch_grad<DT, TEACHER>(ctx, s, g, n);
        });
    });
}

}  // namespace

void launch_token_logprobs(lg_ctx* ctx, hipStream_t s, const LogprobArgs& a) {
    a.dtype == LG_DTYPE_F32   ? logprobs_of<LG_DTYPE_F32>(ctx, s, a)
    : a.dtype == LG_DTYPE_F16 ? logprobs_of<LG_DTYPE_F16>(ctx, s, a)
                              : logprobs_of<LG_DTYPE_BF16>(ctx, s, a);
}

void launch_token_logprobs_backward(lg_ctx* ctx, hipStream_t s, const LogprobBackArgs& a) {
    a.dtype == LG_DTYPE_F32   ? back_of<LG_DTYPE_F32>(ctx, s, a)
    : a.dtype == LG_DTYPE_F16 ? back_of<LG_DTYPE_F16>(ctx, s, a)
                              : back_of<LG_DTYPE_BF16>(ctx, s, a);
}

void launch_distill_grad(lg_ctx* ctx, hipStream_t s, const DistillArgs& a) {
    a.dtype == LG_DTYPE_F32   ? distill_of<LG_DTYPE_F32>(ctx, s, a)
    : a.dtype == LG_DTYPE_F16 ? distill_of<LG_DTYPE_F16>(ctx, s, a)
                              : distill_of<LG_DTYPE_BF16>(ctx, s, a);
}

}  // namespace lg
