// Scoring of class distributions and distillation from a teacher's top alternatives, each with its gradient.
//
// A tensor of logits is rows x classes; z are the logits of a row, y = z / T, c = log2(e) / T.
//   score    lse = log sum_v e^{y_v};  logprob = y_t - lse;  H = -sum_v p_v log p_v;  the K largest classes (ties: the lowest index)
//   distill  the teacher's list (index_k, t_k) per row, t_k = log probabilities:  L = T^2 [ sum_k p_k (log p_k - log q_{index_k})
//            + r (log r - log q_rest) ],  q = softmax(y);  p = softmax_K(t) and r = 0, or (tail) p_k = e^{t_k}, r = 1 - sum p and
//            q_rest the probability of the classes that are not listed
//
// Two families.  Rows of more than COL_MAX contiguous classes: a group of G threads (a wave, or a block) streams a row with the running
// maximum and sums of an online softmax; few long rows are cut into segments whose partial results a second kernel joins.  Short rows, or
// rows whose classes lie at a stride (NCDHW logits of a head): one thread per row holds all classes in registers.
// Sums are float32 per thread and across threads; what cancels (a row's few scalars, 1 - sum p) is combined in float64.
#include "common.h"
#include <algorithm>
#include <type_traits>

namespace mica {

namespace {

typedef unsigned long long u64;
typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef uint4v uint4u __attribute__((aligned(2)));          // 16 bytes at the alignment of an element: one dwordx4 access (unaligned access mode)

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;
constexpr float NEG_BIG = -1.0e30f;                          // stands for -inf where a product with 0 has to stay 0

struct bf16_t { unsigned short u; };
struct f16_t { _Float16 h; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __builtin_bit_cast(float, (unsigned)x.u << 16); }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x.h; }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) { return {__builtin_bit_cast(unsigned short, (__bf16)x)}; }      // to nearest, ties to even
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float x) { return {(_Float16)x}; }

// Which accesses bypass the caches (ONCE), by the size of the logits.  ONCE_STORE beyond 64 MB: what a gradient's stores would push out is
// worth more to whoever runs next (gradient of 4096 x 32000 bf16 117 -> 94 us, 1999 x 65537 f16 114 -> 92).  ONCE_BOTH, where the kernel does
// not read a row twice, beyond 256 MB, the Infinity Cache, if all rows begin on 16 bytes: 4096 x 128000 bf16 scores 196 -> 176 us, loss 201 ->
// 174, 8192 x 16384 f32 106 -> 92, a gradient the same (440); at 262 MB nothing gained, and lost where a later pass would have found the rows
// cached, or where neighbouring lanes share the lines of unaligned vectors (2048 x 50001 f16 66 -> 75 us).
enum { ONCE_NONE, ONCE_STORE, ONCE_BOTH };
template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };

template <typename T> __device__ __forceinline__ uint4v load_raw(const T* p) { return *reinterpret_cast<const uint4u*>(p); }
template <bool ONCE, typename T> __device__ __forceinline__ uint4v load_raw(const T* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const uint4u*>(p));
    else return load_raw(p);
}
// (the whole vector is cast at once: a bit cast of one element of an ext_vector reads element 0)
__device__ __forceinline__ void unpack(uint4v q, float (&f)[4], float*) {
    const floatx4 v = __builtin_bit_cast(floatx4, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = v[j];
}
__device__ __forceinline__ void unpack(uint4v q, float (&f)[8], bf16_t*) {
    const uint4v hi = q & 0xFFFF0000u, lo = q << 16;
    const floatx4 a = __builtin_bit_cast(floatx4, lo), b = __builtin_bit_cast(floatx4, hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = a[j];
        f[2 * j + 1] = b[j];
    }
}
__device__ __forceinline__ void unpack(uint4v q, float (&f)[8], f16_t*) {
    const half8 h = __builtin_bit_cast(half8, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)h[j];
}
// the elements of a raw vector that b names become -inf
__device__ __forceinline__ uint4v raw_drop(uint4v q, unsigned b, float*) {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = (b >> j) & 1u ? 0xFF800000u : q[j];
    return q;
}
template <typename T> __device__ __forceinline__ uint4v raw_drop(uint4v q, unsigned b, T*) {
    constexpr unsigned inf = std::is_same<T, bf16_t>::value ? 0xFF80u : 0xFC00u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[j] = (b >> (2 * j)) & 1u ? (q[j] & 0xFFFF0000u) | inf : q[j];
        q[j] = (b >> (2 * j + 1)) & 1u ? (q[j] & 0xFFFFu) | (inf << 16) : q[j];
    }
    return q;
}
template <typename T> __device__ __forceinline__ uint4v raw_neg_inf();
template <> __device__ __forceinline__ uint4v raw_neg_inf<float>() { return 0xFF800000u; }
template <> __device__ __forceinline__ uint4v raw_neg_inf<bf16_t>() { return 0xFF80FF80u; }
template <> __device__ __forceinline__ uint4v raw_neg_inf<f16_t>() { return 0xFC00FC00u; }
template <bool ONCE, typename T, int N> __device__ __forceinline__ void store_vec(T* p, const float (&f)[N]) {
    struct alignas(16) { T t[N]; } o;
#pragma unroll
    for (int j = 0; j < N; ++j) o.t[j] = from_f32<T>(f[j]);
    if constexpr (ONCE) __builtin_nontemporal_store(__builtin_bit_cast(uint4v, o), reinterpret_cast<uint4u*>(p));
    else *reinterpret_cast<uint4u*>(p) = __builtin_bit_cast(uint4v, o);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- order keys: larger key = larger value; -0 = +0, NaN below every number (with -inf) --------------------------------------------
__device__ __forceinline__ unsigned order_key(float z) {
    z = z + 0.0f;
    const unsigned u = __builtin_bit_cast(unsigned, z);
    return z != z ? 0x007FFFFFu : (u ^ ((unsigned)((int)u >> 31) | 0x80000000u));
}
__device__ __forceinline__ float key_value(unsigned k) {
    return __builtin_bit_cast(float, (k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ u64 make_key(unsigned o, unsigned index) { return ((u64)o << 32) | (0xFFFFFFFFu - index); }
__device__ __forceinline__ unsigned key_index(u64 k) { return 0xFFFFFFFFu - (unsigned)k; }

// ---- exchange between the lanes of a wave, on the vector ALU (no LDS round trip) ---------------------------------------------------------
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) { return __builtin_amdgcn_update_dpp(0u, v, CTRL, 0xF, 0xF, true); }
// the value of lane ^ O
template <int O> __device__ __forceinline__ unsigned lane_xor(unsigned v) {
    if constexpr (O == 1) return dpp<0xB1>(v);                       // quad_perm 1 0 3 2
    else if constexpr (O == 2) return dpp<0x4E>(v);                  // quad_perm 2 3 0 1
    else if constexpr (O == 4) return dpp<0x1B>(dpp<0x141>(v));      // half-row mirror (^ 7), quad_perm 3 2 1 0 (^ 3)
    else if constexpr (O == 8) return dpp<0x128>(v);                 // row rotate by 8
    else if constexpr (O == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? r[0] : r[1];
    }
}
template <int O> __device__ __forceinline__ float lane_xor(float v) { return __builtin_bit_cast(float, lane_xor<O>(__builtin_bit_cast(unsigned, v))); }
template <int O> __device__ __forceinline__ u64 lane_xor(u64 v) { return ((u64)lane_xor<O>((unsigned)(v >> 32)) << 32) | lane_xor<O>((unsigned)v); }
template <int O> __device__ __forceinline__ double lane_xor(double v) { return __builtin_bit_cast(double, lane_xor<O>(__builtin_bit_cast(u64, v))); }

template <typename F, typename Op> __device__ __forceinline__ F wave_all(F v, Op op) {      // the same value in every lane
    v = op(v, lane_xor<1>(v));
    v = op(v, lane_xor<2>(v));
    v = op(v, lane_xor<4>(v));
    v = op(v, lane_xor<8>(v));
    v = op(v, lane_xor<16>(v));
    return op(v, lane_xor<32>(v));
}
__device__ __forceinline__ float wave_max(float v) { return wave_all(v, [](float a, float b) { return fmaxf(a, b); }); }
template <typename F> __device__ __forceinline__ F wave_sum(F v) { return wave_all(v, [](F a, F b) { return a + b; }); }

__device__ __forceinline__ void wave_sync() {                       // LDS written by some lanes of a wave, read by others
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}
template <int G> __device__ __forceinline__ void group_sync() {
    if (G == 64) wave_sync();
    else __syncthreads();
}

// ---- the 64 largest keys of a wave: one per lane, descending ------------------------------------------------------------------------
template <int O> __device__ __forceinline__ u64 cmp_exchange(u64 v, bool take_max) {
    const u64 w = lane_xor<O>(v);
    return (v > w) == take_max ? v : w;
}
// a bitonic sequence -> descending, or ascending
template <bool DESC> __device__ __forceinline__ u64 bitonic_merge64(u64 v, int lane) {
    v = cmp_exchange<32>(v, ((lane & 32) == 0) == DESC);
    v = cmp_exchange<16>(v, ((lane & 16) == 0) == DESC);
    v = cmp_exchange<8>(v, ((lane & 8) == 0) == DESC);
    v = cmp_exchange<4>(v, ((lane & 4) == 0) == DESC);
    v = cmp_exchange<2>(v, ((lane & 2) == 0) == DESC);
    return cmp_exchange<1>(v, ((lane & 1) == 0) == DESC);
}
template <bool DESC> __device__ __forceinline__ u64 sort64(u64 v, int lane) {
#define MICA_SORT_STEP(k, o) v = cmp_exchange<o>(v, ((lane & (o)) == 0) == ((lane & (k)) == 0))
    MICA_SORT_STEP(2, 1);
    MICA_SORT_STEP(4, 2); MICA_SORT_STEP(4, 1);
    MICA_SORT_STEP(8, 4); MICA_SORT_STEP(8, 2); MICA_SORT_STEP(8, 1);
    MICA_SORT_STEP(16, 8); MICA_SORT_STEP(16, 4); MICA_SORT_STEP(16, 2); MICA_SORT_STEP(16, 1);
    MICA_SORT_STEP(32, 16); MICA_SORT_STEP(32, 8); MICA_SORT_STEP(32, 4); MICA_SORT_STEP(32, 2); MICA_SORT_STEP(32, 1);
#undef MICA_SORT_STEP
    return bitonic_merge64<DESC>(v, lane);
}
// a descending, b ascending: the 64 largest of both, descending
__device__ __forceinline__ u64 merge_top64(u64 a, u64 b, int lane) { return bitonic_merge64<true>(a > b ? a : b, lane); }
__device__ __forceinline__ u64 lane_key(u64 v, int l) {             // of a lane known to all
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)v, l), hi = __builtin_amdgcn_readlane((unsigned)(v >> 32), l);
    return ((u64)hi << 32) | lo;
}

// ---- online softmax of one thread -----------------------------------------------------------------------------------------------------
// m: running maximum;  s = sum 2^{z c - R}, w = sum 2^{z c - R} (z c - R) with the reference R = m c rounded to float32: one fma per logit.
// R's rounding, up to half a step of R, is part of every exponent; it cancels, because whoever reads s uses the same R (ref_step(),
// log_sum()), as long as it is small itself.  So beyond |R| = REF_MAX (rounding 1/16; rows masked throughout with -1e9, say) the sums are
// relative to m c itself and the exponents (z - m) c: two instructions.  That is asked of the thread's maximum, at every one that it passes.
constexpr float REF_MAX = 1048576.0f;
constexpr float REF_STEP = 256.0f;                           // 2^-REF_STEP is 0
__device__ __forceinline__ float reference(float m, float c) {
#pragma clang fp contract(off)
    return m * c;
}
__device__ __forceinline__ bool ref_near(float R) { return fabsf(R) <= REF_MAX; }      // not for an infinite maximum
// exponent of the maximum itself
__device__ __forceinline__ float ref_residue(float m, float c) {
    const float R = reference(m, c);
    return ref_near(R) ? fmaf(m, c, -R) : 0.f;
}
// exponent between the references of two maxima, old <= now; -inf - -inf and the like end at NEG_BIG (with empty sums)
__device__ __forceinline__ float ref_step(float old, float now, float c) {
#pragma clang fp contract(off)
    return fmaxf((old - now) * c + (ref_residue(now, c) - ref_residue(old, c)), NEG_BIG);
}
// log of sum_v e^{(z_v - m) / T}; -inf for an empty row
__device__ __forceinline__ double log_sum(float m, double s, float c) { return log(s) - (double)ref_residue(m, c) * LN2; }
struct Online {
    float m = -INFINITY, s = 0.f, w = 0.f;
    // to a maximum >= m
    __device__ __forceinline__ void rescale(float mn, float c) {
        const float d = ref_step(m, mn, c), a = exp2_hw(d);
        if (m == -INFINITY) {                                // nothing so far, or NaN only
            w = s;
        } else {
            w = a * fmaf(s, d, w);
            s *= a;
        }
        m = mn;
    }
    __device__ __forceinline__ void join(Online b, float c) {
        const float mn = fmaxf(m, b.m);
        rescale(mn, c);
        b.rescale(mn, c);
        s += b.s;
        w += b.w;
    }
    // N logits, vmax their maximum (never NaN).  All lanes of a wave call it together.
    template <int N, bool ENT> __device__ __forceinline__ void add(const float (&f)[N], float vmax, float c) {
        const float mn = fmaxf(m, vmax), R = reference(mn, c), old = reference(m, c);
        // some lane's maximum is -inf or of large magnitude, or may have been so while its sums still count
        if (__builtin_expect(__any(!(fabsf(R) <= REF_MAX - REF_STEP)), 0)) {
            rescale(mn, c);
            const float ref = ref_near(R) ? R : 0.f, sub = ref_near(R) || mn == -INFINITY ? 0.f : mn;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float x = fmaf(f[j] - sub, c, -ref);
                const float e = exp2_hw(x);
                s += e;
                if (ENT) w = fmaf(e, fmaxf(x, NEG_BIG), w);
            }
            return;
        }
        const float d = fmaxf(old - R, NEG_BIG);
        const float a = exp2_hw(d);
        if (ENT) w = a * fmaf(s, d, w);
        s *= a;
        m = mn;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float x = fmaf(f[j], c, -R);
            const float e = exp2_hw(x);
            s += e;
            if (ENT) w = fmaf(e, fmaxf(x, NEG_BIG), w);
        }
    }
};
// the joined sums of a wave, in every lane
__device__ __forceinline__ Online wave_join(Online o, float c) {
    o.rescale(wave_max(o.m), c);
    o.s = wave_sum(o.s);
    o.w = wave_sum(o.w);
    return o;
}
struct Partial { float m, s, w, unused; };                 // of a wave, or of a segment of a row
// the joined sums of a group, in every thread (`part`: one entry per wave of the block)
template <int G> __device__ __forceinline__ Online group_join(Online o, float c, Partial* part) {
    o = wave_join(o, c);
    if (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = {o.m, o.s, o.w, 0.f};
        __syncthreads();
        float m = part[0].m;
#pragma unroll
        for (int i = 1; i < G / 64; ++i) m = fmaxf(m, part[i].m);
        o = Online();
        o.m = m;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) {
            Online b;
            b.m = part[i].m; b.s = part[i].s; b.w = part[i].w;
            b.rescale(m, c);
            o.s += b.s;
            o.w += b.w;
        }
    }
    return o;
}

template <int N> __device__ __forceinline__ float max_of(const float (&f)[N]) {
    float v = -INFINITY;                                       // never NaN
#pragma unroll
    for (int j = 0; j < N; ++j) v = fmaxf(v, f[j]);
    return v;
}

__device__ __forceinline__ int64_t load_int(const void* p, int64_t i, int bytes) {
    return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ float load_float(const void* p, int64_t i, int dtype) {
    if (dtype == MICA_F32) return static_cast<const float*>(p)[i];
    if (dtype == MICA_BF16) return to_f32(static_cast<const bf16_t*>(p)[i]);
    return to_f32(static_cast<const f16_t*>(p)[i]);
}

// where row r begins, and where entry (r, k) of a [.., K] list lies: K last, or K in front of the inner rows
struct RowPos { int64_t outer, inner; };
__device__ __forceinline__ RowPos row_pos(const LogitsView& v, int64_t r) {
    if (v.outer == 1) return {0, r};
    const unsigned o = (unsigned)r / (unsigned)v.inner;                       // rows < 2^31
    return {o, r - (int64_t)o * v.inner};
}
__device__ __forceinline__ int64_t row_start(const LogitsView& v, RowPos p) { return p.outer * v.so + p.inner * v.si; }
struct ListPos { int64_t base, stride; };
__device__ __forceinline__ ListPos list_pos(const LogitsView& v, RowPos p, int64_t r, int64_t k) {
    return v.class_last ? ListPos{r * k, 1} : ListPos{p.outer * k * v.inner + p.inner, v.inner};
}

// ========================================================================================================================================
// rows of many classes
// ========================================================================================================================================
constexpr int UNROLL = 4;

// Vector `vec` of the n classes at z, raw: the last one, if n does not fill it, is read from z + n - N with the classes in front of it
// dropped (they lie in this row or, in a later segment, in the one before), so its class nfull N + i is element i + edge_shift.
template <typename T> __device__ __forceinline__ int edge_shift(int n, int vec) {
    constexpr int N = Vec<T>::N;
    return vec == n / N ? N - n % N : 0;
}
template <typename T> __device__ __forceinline__ uint4v load_vec(const T* __restrict__ z, int n, int vec) {
    constexpr int N = Vec<T>::N;
    uint4v q = raw_neg_inf<T>();
    if (vec < n / N) q = load_raw(z + (int64_t)vec * N);
    else if (vec * N < n) q = raw_drop(load_raw(z + (n - N)), (1u << (N - n % N)) - 1u, (T*)nullptr);
    return q;
}
// Streams the n classes at z: f(raw[U], i) for U 16-byte vectors of this thread at a time (vector i + u G is the u-th), with the
// next ones on their way; the last, partial round vector by vector: g(values[N], vector), classes beyond n = -inf.  All threads of the
// group make the same calls, g also for vectors that lie beyond n.
template <typename T, int G, int U, int ONCE, typename F, typename H> __device__ __forceinline__ void stream_row(const T* __restrict__ z, int n, int tid, F&& f, H&& g) {
    constexpr int N = Vec<T>::N;
    const int rounds = n / N / (U * G);                    // of whole vectors only
    const bool more = rounds * U * G * N < n;
    uint4v q[U];
    const auto load = [&](int it) {
        if (it < rounds) {
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = load_raw<ONCE == ONCE_BOTH>(z + (int64_t)(tid + (it * U + u) * G) * N);
        } else if (more) {
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = load_vec(z, n, tid + (it * U + u) * G);
        }
    };
    load(0);
    for (int it = 0; it < rounds; ++it) {
        uint4v now[U];
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = q[u];
        load(it + 1);
        f(now, tid + it * U * G);
    }
    if (more) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (rounds * U + u) * G;
            if (i * N >= n) break;                              // of the whole group
            float v[N];
            unpack(q[u], v, (T*)nullptr);
            g(v, i + tid);
        }
    }
}

// The K <= 64 largest of a group's row.  While streaming, every thread notes its largest value and the vector that held it first.  Of
// these (value, position) pairs each wave takes its ceil(K / waves)-th largest; the smallest of those bounds the K-th largest element
// from below, so only threads at or above the bound can own one of the K.  A long row is noted in PARTS stretches, and only the stretches
// at or above the bound are read once more (about K / (PARTS G) of the row; 4096 x 128000 bf16, K = 20: 272 us with one stretch, 227 with
// four) and what passes the bound is sorted, one key per lane.  More than 64 pass only for K near 64 or in unusual data (many equal
// values, everything large in one place); then every wave merges its share, 64 keys at a time, into a sorted list.  Exact for any data;
// ties and -inf order by index.
struct TopScratch {             // LDS of one wave
    u64 list[64];
    u64 buf[128];
};
struct TopShared { u64 bound[4]; int owners_n, passed; };
constexpr int PARTS = 4;
// what a thread notes: its best of each stretch (per_part rounds of UNROLL vectors; the last one takes the rest)
struct TopNote {
    u64 key[PARTS];
    float best;
    int best_at, part, left;
    bool any;
    __device__ __forceinline__ void start(int per_part) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) key[i] = 0;
        best = -INFINITY;
        best_at = part = 0;
        left = per_part;
        any = false;
    }
    __device__ __forceinline__ void see(float vm, int at) {
        if (vm > best || !any) { best = vm; best_at = at; }
        any = true;
    }
    __device__ __forceinline__ void close() {                   // the stretch ends
        const u64 k = any ? make_key(order_key(best), (unsigned)best_at) : 0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) key[i] = i == part ? k : key[i];
        best = -INFINITY;
        any = false;
    }
    __device__ __forceinline__ void round_done(int per_part) {  // the same in all threads of a group
        if (--left == 0 && part < PARTS - 1) {
            close();
            ++part;
            left = per_part;
        }
    }
};
template <typename T, int G, int U> __device__ __forceinline__ int rounds_per_part(int n) {
    const int rounds = n / Vec<T>::N / (U * G);
    return rounds < PARTS ? 1 : rounds / PARTS;
}
template <typename T, int G, int U>
__device__ __forceinline__ u64 group_top(const T* __restrict__ z, int n, unsigned index0, int k, const TopNote& note, TopScratch* sc, int* owners,
                                         TopShared* sh) {
    constexpr int N = Vec<T>::N, NW = G / 64;
    const int tid = G == 64 ? (threadIdx.x & 63) : threadIdx.x, lane = threadIdx.x & 63, w = G == 64 ? 0 : threadIdx.x >> 6;
    u64 mine = note.key[0];
#pragma unroll
    for (int i = 1; i < PARTS; ++i) mine = note.key[i] > mine ? note.key[i] : mine;
    // waves whose threads all have a class share the K; with none, everything passes
    const int whole = NW == 1 ? 1 : (n / N / 64 < NW ? n / N / 64 : NW);
    const int nth = whole == 0 ? 0 : (k + whole - 1) / whole;
    u64 bound = 0;
    if (nth > 4) bound = lane_key(sort64<true>(mine, lane), nth - 1);
    else {                                                      // a maximum costs a fifth of a sort
        u64 left = mine;
        for (int i = 0; i < nth; ++i) {
            bound = wave_all(left, [](u64 a, u64 b) { return a > b ? a : b; });
            left = left == bound ? 0 : left;
        }
        bound = lane_key(bound, 0);
    }
    int count;
    if (NW > 1) {
        if (lane == 0) sh->bound[w] = bound;
        if (threadIdx.x == 0) sh->owners_n = sh->passed = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i)
            if (i < whole) bound = i == 0 || sh->bound[i] < bound ? sh->bound[i] : bound;
        bound = lane_key(bound, 0);
#pragma unroll
        for (int i = 0; i < PARTS; ++i)                         // the order of the owners does not change the result
            if (note.key[i] != 0 && note.key[i] >= bound) owners[atomicAdd(&sh->owners_n, 1)] = i * G + tid;
        __syncthreads();
        count = __builtin_amdgcn_readfirstlane(sh->owners_n);       // scalar: what follows branches for the whole block
    } else {
        count = 0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const bool own = note.key[i] != 0 && note.key[i] >= bound;
            const u64 b = __ballot(own);
            if (own) owners[count + __popcll(b & ((1ull << lane) - 1))] = i * G + tid;
            count += __popcll(b);
        }
        wave_sync();
    }
    const float bound_value = key_value((unsigned)(bound >> 32));       // (of 0: NaN, below which nothing is)
    const int nvec = (n + N - 1) / N, rounds = nvec / (U * G) + 1, per_part = rounds_per_part<T, G, U>(n);
    // the longest stretch, in vectors of one thread: the last one
    const int per = (rounds - (PARTS - 1) * per_part > per_part ? rounds - (PARTS - 1) * per_part : per_part) * U;
    const int total = count * per;
    // take(passes, key), by whole waves, for the classes the owners hold, at least those that pass
    const auto scan = [&](auto&& take) {
        for (int p0 = 0; p0 < total; p0 += G) {
            const int p = p0 + tid;
            int vec = nvec;
            if (p < total) {
                const int own = owners[p % count], part = own / G, i = p / count;       // the i-th vector of the stretch
                if (part == PARTS - 1 || i < per_part * U) vec = own % G + (part * per_part * U + i) * G;
                if (vec > nvec) vec = nvec;
            }
            const int shift = edge_shift<T>(n, vec);
            float v[N];
            unpack(load_vec(z, n, vec), v, (T*)nullptr);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (!__any(!(v[j] < bound_value))) continue;    // NaN counts as -inf
                const int at = vec * N + j - shift;
                const unsigned o = order_key(v[j]);
                take(vec < nvec && j >= shift && make_key(o, (unsigned)(vec * N)) >= bound, make_key(o, (unsigned)at));
            }
        }
    };
    u64 list = 0;
    bool few = false;
    if (NW > 1) {
        scan([&](bool pass, u64 key) {
            if (pass) {
                const int i = atomicAdd(&sh->passed, 1);
                if (i < 64) sc[0].buf[i] = key;
            }
        });
        __syncthreads();
        const int passed = __builtin_amdgcn_readfirstlane(sh->passed);
        few = passed <= 64;
        if (few) {
            if (w == 0) list = sort64<true>(lane < passed ? sc[0].buf[lane] : 0, lane);
        } else {
            __syncthreads();                                    // buf is about to be written again
        }
    }
    if (!few) {
        u64 floor_key = 0;
        int pending = 0;
        scan([&](bool pass0, u64 key) {
            const bool pass = pass0 && key > floor_key;
            const u64 b = __ballot(pass);
            if (b == 0) return;
            if (pass) sc[w].buf[pending + __popcll(b & ((1ull << lane) - 1))] = key;
            pending += __popcll(b);
            wave_sync();
            if (pending >= 64) {
                const u64 now = sc[w].buf[lane], rest = sc[w].buf[64 + lane];
                wave_sync();
                sc[w].buf[lane] = rest;
                wave_sync();
                pending -= 64;
                list = merge_top64(list, sort64<false>(now, lane), lane);
                floor_key = lane_key(list, k - 1);
            }
        });
        if (pending > 0) list = merge_top64(list, sort64<false>(lane < pending ? sc[w].buf[lane] : 0, lane), lane);
        if (NW > 1) {
            sc[w].list[lane] = list;
            __syncthreads();
            if (w == 0) {
#pragma unroll
                for (int i = 1; i < NW; ++i) list = merge_top64(list, sc[i].list[63 - lane], lane);
            }
        }
    }
    // (of wave 0) classes are numbered within the segment so far
    return list == 0 ? 0 : ((list & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (key_index(list) + index0)));
}

// -inf is kept for rows without a class: a log sum of -3.4e38 / T, T < 1, is the lowest value
__device__ __forceinline__ float finite(float x) { return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f); }
// a row's results from its joined sums; one thread
struct ScoreOut {
    const void* tokens;
    int token_bytes;
    int64_t ignore;
    float* logprob;
    float* entropy;
    float* lse;
    float* top_logprob;
    int* top_index;
    int top;
    float c, inv_t;
    float* aux;         // [2][rows], nullable: maximum and sum of e^{(z - maximum) / T}, for the gradient
    int64_t rows;
};
// L: the type the row's scalars are combined in
template <typename L> __device__ __forceinline__ float class_logprob(float z, float m, L log_s, float inv_t) {
    const float lp = m == -INFINITY ? (log_s != log_s ? (float)log_s : -INFINITY) : (float)((L)(z - m) * inv_t - log_s);
    return lp > 0.f ? 0.f : lp;                                 // a sum that rounded to just below 1
}
template <typename T, typename L>
__device__ __forceinline__ void write_row(const ScoreOut& o, const T* __restrict__ z, int64_t sc, int64_t classes, int64_t r, float m, float s, float w,
                                          L log_s) {
    o.lse[r] = s != s ? s : (m == -INFINITY ? -INFINITY : finite((float)((L)m * o.inv_t + log_s)));
    // log2 s - w / s in the units of R cancels nothing: both parts of the entropy are >= 0 up to rounding
    const L log2_s = sizeof(L) == 8 ? (L)log2((double)s) : (L)log2f(s);
    const float h = s == 0.f ? 0.f : (float)((L)LN2 * (log2_s - (L)w / (L)s));
    o.entropy[r] = h < 0.f ? 0.f : h;
    if (o.aux) {
        o.aux[r] = m;
        o.aux[o.rows + r] = s * exp2_hw(-ref_residue(m, o.c));
    }
    if (o.logprob) {
        const int64_t t = load_int(o.tokens, r, o.token_bytes);
        float lp;
        if (t == o.ignore) lp = 0.f;
        else if (t < 0 || t >= classes) lp = NAN;
        else lp = s != s ? s : class_logprob<L>(to_f32(z[t * sc]), m, log_s, o.inv_t);
        o.logprob[r] = lp;
    }
}
__device__ __forceinline__ void write_top(const ScoreOut& o, const LogitsView& v, RowPos p, int64_t r, u64 key, int lane, float m, float s, double log_s) {
    if (lane < o.top) {
        const ListPos l = list_pos(v, p, r, o.top);
        o.top_logprob[l.base + lane * l.stride] = s != s ? s : class_logprob<double>(key_value((unsigned)(key >> 32)), m, log_s, o.inv_t);
        o.top_index[l.base + lane * l.stride] = (int)key_index(key);
    }
}

// One read of the logits.  HBM-bound without alternatives: 4096 x 128000 bf16 175 us = 6.0 TB/s (a bare read of it 152-175 us), 7.6
// instructions and one exponential per logit, half of the issue slots.  With alternatives the selection behind the stream is not hidden
// by the other blocks of the CU: 227 us for K = 20.  Two vectors at a time then, which leaves registers for six blocks.  (The waves per SIMD
// in the bounds here and of the other kernels are what the stream's own registers allow; the path of far rows would cost one wave.)
template <typename T, int G, bool TOP, int ONCE>
__global__ __launch_bounds__(256, sizeof(T) == 4 && !TOP ? 8 : 6) void score_row_kernel(LogitsView v, int64_t rows, ScoreOut o, int segments, int seg_len, Partial* __restrict__ part,
                                                        u64* __restrict__ part_top) {
    constexpr int N = Vec<T>::N, NW = G / 64, GROUPS = 256 / G, U = TOP ? 2 : UNROLL;
    __shared__ Partial waves[4];
    __shared__ TopScratch top_sc[TOP ? 4 : 1];
    __shared__ int owners[TOP ? 256 * PARTS : 1];
    __shared__ TopShared top_sh;
    const int g = threadIdx.x / G, tid = threadIdx.x % G, lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + g;
    if (item >= rows * segments) return;                   // whole waves; with G = 256 the grid is exact
    const int64_t r = segments == 1 ? item : item / segments;
    const int seg = segments == 1 ? 0 : (int)(item % segments);
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    const int first = seg * seg_len;
    const int n = (int)(v.classes - first < seg_len ? v.classes - first : seg_len);
    Online on;
    TopNote note;
    const int per_part = rounds_per_part<T, G, U>(n);
    if (TOP) note.start(per_part);
    stream_row<T, G, U, ONCE>(
        z + first, n, tid,
        [&](const uint4v(&q)[U], int i) {
            float f[U * N], vm = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[N];
                unpack(q[u], x, (T*)nullptr);
                const float mu = max_of(x);
                if (TOP) note.see(mu, (i + u * G) * N);
                vm = fmaxf(vm, mu);
#pragma unroll
                for (int j = 0; j < N; ++j) f[u * N + j] = x[j];
            }
            if (TOP) note.round_done(per_part);
            on.add<U * N, true>(f, vm, o.c);
        },
        [&](const float(&f)[N], int vec) {
            const float vm = max_of(f);
            if (TOP && vec * N < n) note.see(vm, vec * N);
            on.add<N, true>(f, vm, o.c);
        });
    on = group_join<G>(on, o.c, waves);
    u64 key = 0;
    if (TOP) {
        note.close();
        key = group_top<T, G, U>(z + first, n, (unsigned)first, o.top, note, NW == 1 ? &top_sc[g] : top_sc, &owners[g * G * PARTS], &top_sh);
    }
    if (segments == 1) {
        if (tid < 64) {
            const double log_s = log_sum(on.m, on.s, o.c);        // s is about 1 or more unless the row is empty (0) or holds NaN
            if (lane == 0) write_row<T, double>(o, z, 1, v.classes, r, on.m, on.s, on.w, log_s);
            if (TOP) write_top(o, v, p, r, key, lane, on.m, on.s, log_s);
        }
    } else {
        if (tid == 0) part[item] = {on.m, on.s, on.w, 0.f};
        if (TOP && tid < o.top) part_top[item * 64 + tid] = key;
    }
}

// joins the segments of a row: a block of 16 waves
constexpr int JOIN = 1024;
__device__ __forceinline__ Online join_segments(const Partial* __restrict__ part, int segments, float c) {      // one wave; in every lane
    Online on;
    for (int i = threadIdx.x & 63; i < segments; i += 64) {
        const Partial q = part[i];
        Online b;
        b.m = q.m; b.s = q.s; b.w = q.w;
        on.join(b, c);
    }
    return wave_join(on, c);
}
template <typename T, bool TOP>
__global__ __launch_bounds__(TOP ? JOIN : 64) void score_join_kernel(LogitsView v, ScoreOut o, int segments, const Partial* __restrict__ part,
                                                                     const u64* __restrict__ part_top) {
    __shared__ u64 lists[TOP ? JOIN / 64 : 1][64];
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    u64 list = 0;
    if (TOP) {                                                      // every wave merges its share, then a tree over the waves
        for (int i = w; i < segments; i += JOIN / 64) {
            const u64* q = part_top + (r * segments + i) * 64;
            list = merge_top64(list, 63 - lane < o.top ? q[63 - lane] : 0, lane);
        }
        lists[w][lane] = list;
#pragma unroll
        for (int h = JOIN / 128; h > 0; h >>= 1) {
            __syncthreads();
            if (w < h) {
                list = merge_top64(list, lists[w + h][63 - lane], lane);
                lists[w][lane] = list;                              // read by nobody in this round: waves w + h >= h read nothing below h
            }
        }
    }
    if (w > (TOP ? 1 : 0)) return;
    const Online on = join_segments(part + r * segments, segments, o.c);
    const double log_s = log_sum(on.m, on.s, o.c);
    if (TOP && w == 0) write_top(o, v, p, r, list, lane, on.m, on.s, log_s);
    if (w == (TOP ? 1 : 0) && lane == 0) write_row<T, double>(o, z, 1, v.classes, r, on.m, on.s, on.w, log_s);
}

// ---- gradient of the scores ------------------------------------------------------------------------------------------------------------
// dz_v = (1/T) [ g_lp ([v = t] - p_v) + g_lse p_v - g_H p_v (log p_v + H) ]: one read, one write.  p = 2^d / S with d = (z - m) c, from the
// row's maximum m and sum S apart: a float32 log sum of a row of large magnitude has lost log S (a row of -1e9: all of it).  Streamed rows
// get both from the forward pass, the column kernel has the classes in registers and sums again.  HBM-bound: 4096 x 32000 bf16 94 us = 5.6
// TB/s, above the rate of a copy because the forward pass left part of the logits in the Infinity Cache.
struct ScoreGrad {
    const void* tokens;
    int token_bytes;
    int64_t ignore;
    const float* aux;
    int64_t rows;
    const float* entropy;
    const float* g_logprob;
    const float* g_entropy;
    const float* g_lse;
    float c, inv_t;
};
struct RowGrad {
    float m, c;
    float a;            // coefficient of 2^d
    float b;            // coefficient of 2^d d
    float at_token;     // added at the token
    int64_t token;      // -1: none
    bool empty;
};
__device__ __forceinline__ RowGrad row_grad(const ScoreGrad& o, int64_t classes, int64_t r, float m, float s) {
    RowGrad g;
    g.empty = m == -INFINITY && s == 0.f;
    g.m = m;
    g.c = o.c;
    float glp = 0.f;
    g.token = -1;
    if (o.g_logprob) {
        const int64_t t = load_int(o.tokens, r, o.token_bytes);
        if (t != o.ignore) {
            glp = o.g_logprob[r];
            if (t >= 0 && t < classes) g.token = t;
            else glp = NAN;
        }
    }
    const float ge = o.g_entropy ? o.g_entropy[r] : 0.f, gl = o.g_lse ? o.g_lse[r] : 0.f;
    const float scale = o.inv_t / s;                        // log p + H = d log 2 + (H - log S)
    g.a = (gl - glp - (ge != 0.f ? ge * (o.entropy[r] - logf(s)) : 0.f)) * scale;
    g.b = -ge * (float)LN2 * scale;
    g.at_token = g.empty ? 0.f : glp * o.inv_t;
    return g;
}
__device__ __forceinline__ float grad_value(const RowGrad& g, float z) {
    const float d = (z - g.m) * g.c;
    // (2^d is 0 long before -1024; beyond it only the product with a large b, an entropy's scaled gradient at a small T, would overflow)
    return g.empty ? 0.f : exp2_hw(d) * fmaf(g.b, fmaxf(d, -1024.f), g.a);
}

// what a block of the gradient kernels covers: G threads x UNROLL vectors of one row
template <typename T, int G, int ONCE, typename F>
__device__ __forceinline__ void map_chunk(const T* __restrict__ z, T* __restrict__ out, int first, int64_t classes, int tid, F&& f) {
    constexpr int N = Vec<T>::N;
    uint4v q[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t at = first + (int64_t)(tid + u * G) * N;
        if (at + N <= classes) q[u] = load_raw<ONCE == ONCE_BOTH>(z + at);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t at = first + (int64_t)(tid + u * G) * N;
        if (at + N <= classes) {
            float v[N];
            unpack(q[u], v, (T*)nullptr);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = f(v[j], at + j);
            store_vec<ONCE != ONCE_NONE>(out + at, v);
        } else {
            for (int j = 0; j < N; ++j)
                if (at + j < classes) out[at + j] = from_f32<T>(f(to_f32(z[at + j]), at + j));
        }
    }
}

template <typename T, int G, int ONCE>
__global__ __launch_bounds__(256) void score_grad_row_kernel(LogitsView v, int64_t rows, ScoreGrad o, int chunks, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / G, CHUNK = G * UNROLL * Vec<T>::N;
    const int tid = threadIdx.x % G;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G;
    if (item >= rows * chunks) return;
    const int64_t r = chunks == 1 ? item : item / chunks;
    const int first = chunks == 1 ? 0 : (int)(item % chunks) * CHUNK;
    const RowGrad g = row_grad(o, v.classes, r, o.aux[r], o.aux[o.rows + r]);
    const T* z = static_cast<const T*>(v.p) + row_start(v, row_pos(v, r));
    map_chunk<T, G, ONCE>(z, grad + r * v.classes, first, v.classes, tid, [&](float x, int64_t at) { return grad_value(g, x) + (at == g.token ? g.at_token : 0.f); });
}

// ---- distillation ------------------------------------------------------------------------------------------------------------------------
struct DistillArgs {
    const void* index;
    int index_bytes;
    const void* teacher;
    int teacher_dtype;
    int k;
    int tail;
    float c, t;
    double inv_t;                 // of the few terms that are combined in float64
    const float* weight;          // nullable: rows of weight 0 are skipped
    float* loss;
    float* aux;                   // [4][rows], nullable: RowGradient's m, f, M (tail) or norm, qs
    const float* g_loss;          // gradient kernels
};
// A row's gradient, times T and the upstream gradient: (mass q_rest - r) times the share e^{y} / sum of e^{y} among the classes that are
// not listed, for these (nothing overflows where q_rest is tiny), and mass q - sum p for the listed ones.  Both are kept relative to a
// maximum, not to a log sum: a float32 log sum of a row of the type's lowest values would have lost the number of its classes.
struct RowGradient {
    float m, f;         // not listed: f 2^{z c - R(m)}, or f 2^{(z - m) c} beyond REF_MAX
    float M, qs;        // listed: qs 2^{(z - M) c} - sum p
    float t0, norm;     // log p = (t - t0) - norm: the list's maximum and the log of its sum apart, as an offset of 1e8 would swallow the latter
    __device__ __forceinline__ bool empty() const { return M == -INFINITY; }
};
// The row's list in LDS: index (unused entries -1, no class: INT_MAX), log probability, logit.  Loaded by one wave.
struct ListLds { int* i; float* t; float* z; };
constexpr unsigned LIST_BYTES = 12;                             // of LDS per entry
__device__ __forceinline__ ListLds list_lds(int* base, int k) { return {base, reinterpret_cast<float*>(base + k), reinterpret_cast<float*>(base + 2 * k)}; }
template <typename T>
__device__ __forceinline__ void list_load(const DistillArgs& a, ListPos l, const T* __restrict__ z, int64_t classes, int lane, ListLds d) {
    for (int k = lane; k < a.k; k += 64) {
        const int64_t v = load_int(a.index, l.base + k * l.stride, a.index_bytes);
        const float t = load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype);
        d.i[k] = v < 0 ? -1 : (v >= classes ? 0x7FFFFFFF : (int)v);
        d.t[k] = v < 0 ? -INFINITY : t;
        d.z[k] = v < 0 || v >= classes ? -INFINITY : to_f32(z[v]);
    }
}
// A bit per class, laid out as the stream reads it: class v of vector vec = v / N is bit (vec / G % U) * 8 + v % N of word
// (vec / (U G)) G + vec % G, one word for the U vectors a thread takes at a time.
template <typename T, int G, int U = UNROLL> __host__ __device__ constexpr int mark_words(int n) {
    return ((n + Vec<T>::N - 1) / Vec<T>::N + U * G - 1) / (U * G) * G;
}
template <typename T, int G, int U = UNROLL> __device__ __forceinline__ void mark_listed(const int* idx, int k, int first, int n, unsigned* bits, int tid) {
    constexpr int N = Vec<T>::N;
    for (int i = tid; i < mark_words<T, G, U>(n); i += G) bits[i] = 0;
    group_sync<G>();
    for (int i = tid; i < k; i += G) {
        const int v = idx[i] - first;
        if (idx[i] >= 0 && v >= 0 && v < n) {
            const int vec = v / N;
            atomicOr(&bits[vec / (U * G) * G + vec % G], 1u << (vec / G % U * 8 + v % N));
        }
    }
    group_sync<G>();
}
template <int N> __device__ __forceinline__ void drop_listed(float (&f)[N], unsigned b) {
    if (b) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = (b >> j) & 1u ? -INFINITY : f[j];
    }
}
// the online sums of the classes of a segment, without the listed ones if TAIL
template <typename T, int G, bool TAIL, int U, int ONCE>
__device__ __forceinline__ Online distill_stream(const T* __restrict__ z, int n, int tid, const unsigned* bits, float c) {
    constexpr int N = Vec<T>::N;
    Online on;
    stream_row<T, G, U, ONCE>(
        z, n, tid,
        [&](const uint4v(&q)[U], int i) {
            const unsigned b = TAIL ? bits[i / U / G * G + tid] : 0u;
            float f[U * N], vm = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[N];
                unpack(q[u], x, (T*)nullptr);
                if (TAIL) drop_listed(x, (b >> (8 * u)) & 0xFFu);
                vm = fmaxf(vm, max_of(x));
#pragma unroll
                for (int j = 0; j < N; ++j) f[u * N + j] = x[j];
            }
            on.add<U * N, false>(f, vm, c);
        },
        [&](const float(&f0)[N], int vec) {
            float f[N];
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = f0[j];
            if (TAIL && vec * N < n) drop_listed(f, ((bits[vec / (U * G) * G + vec % G] >> (vec / G % U * 8)) & 0xFFu) << edge_shift<T>(n, vec));
            on.add<N, false>(f, max_of(f), c);
        });
    return on;
}

// the maximum of the list's values, 0 if that is -inf; one wave, in every lane
__device__ __forceinline__ float list_max(const DistillArgs& a, ListLds d, int lane) {
    float t = -INFINITY;
    for (int k = lane; k < a.k; k += 64) t = fmaxf(t, d.t[k]);
    t = wave_max(t);
    return t == -INFINITY ? 0.f : t;
}
// What a row's list says by itself: one wave, in every lane.
struct ListStats {
    double mass;        // sum p: of the renormalised list 1, or 0 if no entry has any; tail: sum of e^t
    float t0;           // the values' maximum (renormalised; of no entry with any probability 0), 0 (tail)
    double norm;        // log of the sum of e^{t - t0} (renormalised; -inf: none has any), 0 (tail)
    double log_sl;      // (tail) log of the listed classes' sum relative to zmax, every class once; -inf: none
    float zmax;
    int bad;            // an index that is no class
};
__device__ __forceinline__ ListStats list_stats(const DistillArgs& a, ListLds d, int lane) {
    ListStats o;
    bool bad = false;
    float tmax = -INFINITY, zmax = -INFINITY;
    for (int k = lane; k < a.k; k += 64) {
        bad |= d.i[k] == 0x7FFFFFFF;
        tmax = fmaxf(tmax, d.t[k]);
        zmax = fmaxf(zmax, d.z[k]);
    }
    o.bad = __any(bad);
    o.zmax = zmax = wave_max(zmax);
    o.log_sl = -INFINITY;
    if (!a.tail) {
        tmax = wave_max(tmax);
        double sum = 0.0;
        for (int k = lane; k < a.k; k += 64)
            if (d.i[k] >= 0) sum += tmax == -INFINITY ? (d.t[k] != d.t[k] ? (double)d.t[k] : 0.0) : exp((double)d.t[k] - tmax);
        sum = wave_sum(sum);
        o.t0 = tmax == -INFINITY ? 0.f : tmax;
        o.norm = tmax == -INFINITY && sum != 0.0 ? sum : log(sum);
        o.mass = sum == 0.0 ? 0.0 : 1.0;
    } else {
        double sl = 0.0, P = 0.0;
        for (int k = lane; k < a.k; k += 64) {
            const int i = d.i[k];
            if (i < 0) continue;
            P += exp((double)d.t[k]);
            bool again = false;
            for (int j = 0; j < k; ++j) again |= d.i[j] == i;
            if (!again) sl += zmax == -INFINITY ? (d.z[k] != d.z[k] ? (double)d.z[k] : 0.0) : (double)exp2_hw((d.z[k] - zmax) * a.c);
        }
        o.log_sl = log(wave_sum(sl));
        o.mass = wave_sum(P);
        o.t0 = 0.f;
        o.norm = 0.0;
    }
    return o;
}
// The row's scalars from its list and the sums over all classes, or over those that are not listed (tail); any thread.  What cancels is
// combined in float64: 1 - sum p, log q_rest = -log(1 + listed sum / rest sum).
struct RowScalars { double M, log_s, rest, log_q_rest, mass; bool invalid; RowGradient g; };     // M, log_s: maximum and log sum of all classes
__device__ __forceinline__ RowScalars row_scalars(const DistillArgs& a, const ListStats& l, float m, float s) {
    RowScalars o;
    const double log_m = log_sum(m, s, a.c);                    // log of the streamed sum relative to m
    o.M = m;
    o.log_s = log_m;
    o.rest = o.log_q_rest = 0.0;
    o.mass = l.mass;
    const bool have_rest = !(s == 0.f);                         // NaN counts
    double factor = o.mass;
    if (a.tail) {
        o.rest = have_rest && l.mass < 1.0 ? 1.0 - l.mass : 0.0;
        o.mass += o.rest;
        if (!have_rest) { o.M = l.zmax; o.log_s = l.log_sl; }
        else if (l.log_sl != -INFINITY) {
            // the two parts of the row's sum, relative to M: the larger one is about 1 or more, which the smaller one's log does not swallow
            o.M = fmaxf(m, l.zmax);
            const double r = ((double)m - o.M) * a.inv_t + log_m, t = ((double)l.zmax - o.M) * a.inv_t + l.log_sl, u = t - r;
            const double v = log1p(exp(-fabs(u)));
            o.log_q_rest = -(fmax(u, 0.0) + v);
            o.log_s = fmax(r, t) + v;
        }
        factor = o.mass * exp(o.log_q_rest) - o.rest;
    }
    // a NaN anywhere, or an index that is no class: loss and gradient of the whole row are NaN
    o.invalid = l.bad || s != s || o.log_s != o.log_s || o.mass != o.mass || l.norm != l.norm;
    o.g.m = a.tail && !have_rest ? 0.f : m;                    // without a tail M itself
    o.g.f = have_rest ? (float)(factor / s) : 0.f;
    o.g.M = (float)o.M;
    o.g.qs = o.M == -INFINITY ? 0.f : (float)(o.mass * exp(-o.log_s));
    o.g.t0 = l.t0;
    o.g.norm = (float)l.norm;
    return o;
}
// the loss; one wave, in every lane
__device__ __forceinline__ float row_loss(const DistillArgs& a, ListLds d, const ListStats& l, const RowScalars& o, int lane) {
    double sum = 0.0;
    for (int k = lane; k < a.k; k += 64) {
        if (d.i[k] < 0) continue;
        const double lp = ((double)d.t[k] - l.t0) - l.norm;
        const double pk = o.mass == 0.0 ? 0.0 : exp(lp);
        const double lq = o.M == -INFINITY ? -INFINITY : ((double)d.z[k] - o.M) * a.inv_t - o.log_s;
        if (!(pk == 0.0)) sum += pk * (lp - lq);
    }
    sum = wave_sum(sum);
    if (o.rest > 0.0) sum += o.rest * (log(o.rest) - o.log_q_rest);
    return o.invalid ? NAN : (float)(sum * a.t * a.t);
}
// loss and aux of a row from its joined sums; one wave, the result in every lane
__device__ __forceinline__ RowGradient finish_row(const DistillArgs& a, ListLds d, float m, float s, int64_t r, int64_t rows, int lane) {
    const ListStats l = list_stats(a, d, lane);
    const RowScalars o = row_scalars(a, l, m, s);
    const float loss = row_loss(a, d, l, o, lane);
    RowGradient q = o.g;
    if (loss != loss) {
        q.f = q.qs = NAN;
        if (q.empty()) q.m = q.M = 0.f;                         // or its gradient would be the empty row's, 0
    }
    if (lane == 0) {
        const float w = a.weight ? a.weight[r] : 1.f;
        a.loss[r] = w == 0.f ? 0.f : loss * w;
        if (a.aux) {
            a.aux[r] = q.m;
            a.aux[rows + r] = q.f;
            a.aux[2 * rows + r] = a.tail ? q.M : q.norm;        // without a tail M = m
            a.aux[3 * rows + r] = q.qs;
        }
    }
    return q;
}

// One read of the logits, a bit of LDS per class to leave out the listed ones (tail; subtracting them afterwards would cancel for every
// good student).  HBM-bound: 4096 x 128000 bf16 174 us = 6.0 TB/s, 185 with the tail and 64 entries; 513 x 32003 15 us, the latency of its steps.
template <typename T, int G, bool TAIL, int ONCE>
__global__ __launch_bounds__(256, (sizeof(T) == 4 ? 7 : 5) + (G == 256)) void distill_row_kernel(LogitsView v, int64_t rows, DistillArgs a, int segments, int seg_len, Partial* __restrict__ part) {
    constexpr int GROUPS = 256 / G;
    extern __shared__ int dyn[];
    __shared__ Partial waves[4];
    const int g = threadIdx.x / G, tid = threadIdx.x % G, lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + g;
    if (item >= rows * segments) return;
    const int64_t r = segments == 1 ? item : item / segments;
    const int seg = segments == 1 ? 0 : (int)(item % segments);
    const int words = TAIL ? mark_words<T, G>(seg_len) : 0;
    const ListLds list = list_lds(dyn + g * (3 * a.k + words), a.k);
    unsigned* bits = reinterpret_cast<unsigned*>(list.z + a.k);
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    const int first = seg * seg_len;
    const int n = (int)(v.classes - first < seg_len ? v.classes - first : seg_len);
    if (tid < 64) list_load(a, list_pos(v, p, r, a.k), z, v.classes, lane, list);
    group_sync<G>();
    if (TAIL) mark_listed<T, G>(list.i, a.k, first, n, bits, tid);
    const Online on = group_join<G>(distill_stream<T, G, TAIL, UNROLL, ONCE>(z + first, n, tid, bits, a.c), a.c, waves);
    if (segments > 1) {
        if (tid == 0) part[item] = {on.m, on.s, 0.f, 0.f};
        return;
    }
    if (tid < 64) (void)finish_row(a, list, on.m, on.s, r, rows, lane);
}
template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(LogitsView v, int64_t rows, DistillArgs a, int segments, const Partial* __restrict__ part) {
    extern __shared__ int dyn[];
    const int64_t r = blockIdx.x;
    const RowPos p = row_pos(v, r);
    const ListLds list = list_lds(dyn, a.k);
    list_load(a, list_pos(v, p, r, a.k), static_cast<const T*>(v.p) + row_start(v, p), v.classes, threadIdx.x, list);
    wave_sync();
    const Online on = join_segments(part + r * segments, segments, a.c);
    (void)finish_row(a, list, on.m, on.s, r, rows, threadIdx.x);
}

// the listed classes of [first, first + n): overwrites what the sweep wrote there; the first mention of a class writes for all of them
template <typename T, int G>
__device__ __forceinline__ void listed_grad(const DistillArgs& a, T* __restrict__ out, ListLds d, int64_t first, int64_t n, RowGradient q, float scale, int tid) {
    for (int k = tid; k < a.k; k += G) {
        const int i = d.i[k];
        if (i < first || i >= first + n || i < 0 || i == 0x7FFFFFFF) continue;
        bool again = false;
        float p = 0.f;
        for (int j = 0; j < a.k; ++j) {
            if (d.i[j] != i) continue;
            again |= j < k;
            p += a.tail ? expf(d.t[j]) : (q.norm == -INFINITY ? 0.f : expf((d.t[j] - q.t0) - q.norm));
        }
        if (!again) out[i] = from_f32<T>(scale * (q.qs * exp2_hw((d.z[k] - q.M) * a.c) - p));
    }
}
// the gradient of a class that is not listed
struct Unlisted {
    float sub, R, f, c;
    bool none;
    __device__ __forceinline__ Unlisted(const DistillArgs& a, const RowGradient& q, float scale) {
        none = q.empty() || scale == 0.f;
        const bool far = !ref_near(reference(q.m, a.c));
        sub = far ? q.m : 0.f;
        R = far || none ? 0.f : reference(q.m, a.c);
        f = none ? 0.f : scale * q.f;
        c = a.c;
    }
    __device__ __forceinline__ float operator()(float z) const { return none ? 0.f : f * exp2_hw(fmaf(z - sub, c, -R)); }
};

// One read, one write: 1999 x 65537 f16 93 us = 5.6 TB/s.
template <typename T, int G, int ONCE>
__global__ __launch_bounds__(256) void distill_grad_row_kernel(LogitsView v, int64_t rows, DistillArgs a, int chunks, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / G, CHUNK = G * UNROLL * Vec<T>::N;
    extern __shared__ int dyn[];
    __shared__ float t0[GROUPS];
    const int g = threadIdx.x / G, tid = threadIdx.x % G;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + g;
    if (item >= rows * chunks) return;
    const int64_t r = chunks == 1 ? item : item / chunks;
    const int first = chunks == 1 ? 0 : (int)(item % chunks) * CHUNK;
    const ListLds list = list_lds(dyn + g * 3 * a.k, a.k);
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    if (tid < 64) {
        list_load(a, list_pos(v, p, r, a.k), z, v.classes, tid, list);
        const float t = a.tail ? 0.f : list_max(a, list, tid);      // of the entries that this lane has written
        if (tid == 0) t0[g] = t;
    }
    T* out = grad + r * v.classes;
    const float w = a.weight ? a.weight[r] : 1.f;
    const float scale = (a.g_loss ? a.g_loss[r] : 1.f) * w * a.t;
    const float x = a.aux[2 * rows + r], m = a.aux[r];
    RowGradient o{m, a.aux[rows + r], a.tail ? x : m, a.aux[3 * rows + r], 0.f, a.tail ? 0.f : x};
    const Unlisted unlisted(a, o, scale);
    map_chunk<T, G, ONCE>(z, out, first, v.classes, tid, [&](float y, int64_t) { return unlisted(y); });
    group_sync<G>();
    o.t0 = t0[g];
    if (!unlisted.none) listed_grad<T, G>(a, out, list, first, CHUNK, o, scale, tid);
}

// Loss and gradient in one kernel: the row is read twice, the second time from cache, and its gradient written.  So that the second
// read finds it there, G is chosen to leave few rows in flight: 2048 / G blocks on a CU (step_group).  4096 x 128000 bf16 495 us = 4.2 TB/s
// of one read and one write; as a call 507, the two-kernel form 547, 256 threads per row 637 (the second read from HBM).  Holding the row in
// the registers of 1024 threads took 562: one block on a CU, nothing to do while it sums.
constexpr int STEP_U = 2;                                       // 64 registers: two blocks of 1024 threads on a CU
template <typename T, int G, bool TAIL, int ONCE>
__global__ __launch_bounds__(G < 256 ? 256 : G, 8) void distill_step_kernel(LogitsView v, int64_t rows, DistillArgs a, T* __restrict__ grad) {
    constexpr int BLOCK = G < 256 ? 256 : G, GROUPS = BLOCK / G, N = Vec<T>::N;
    extern __shared__ int dyn[];
    __shared__ Partial waves[BLOCK / 64];
    __shared__ RowGradient shared_row[GROUPS];
    const int g = threadIdx.x / G, tid = threadIdx.x % G, lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * GROUPS + g;
    if (r >= rows) return;
    const int n = (int)v.classes;
    const int words = TAIL ? mark_words<T, G, STEP_U>(n) : 0;
    const ListLds list = list_lds(dyn + g * (3 * a.k + words), a.k);
    unsigned* bits = reinterpret_cast<unsigned*>(list.z + a.k);
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    T* out = grad + r * v.classes;
    if (tid < 64) list_load(a, list_pos(v, p, r, a.k), z, v.classes, lane, list);
    group_sync<G>();
    if (TAIL) mark_listed<T, G, STEP_U>(list.i, a.k, 0, n, bits, tid);
    const Online on = group_join<G>(distill_stream<T, G, TAIL, STEP_U, ONCE>(z, n, tid, bits, a.c), a.c, waves);
    RowGradient o;
    if (tid < 64) {
        o = finish_row(a, list, on.m, on.s, r, rows, lane);
        if (lane == 0) shared_row[g] = o;
    }
    if (G > 64) {
        __syncthreads();
        o = shared_row[g];
    }
    const float scale = a.t * (a.weight ? a.weight[r] : 1.f);
    const Unlisted unlisted(a, o, scale);
    const auto put = [&](const float(&y)[N], int vec) {
        float d[N];
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] = unlisted(y[j]);
        if (vec < n / N) store_vec<ONCE != ONCE_NONE>(out + (int64_t)vec * N, d);
        else if (vec * N < n) {
            const int shift = edge_shift<T>(n, vec);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j >= shift) out[n - N + j] = from_f32<T>(d[j]);
        }
    };
    stream_row<T, G, STEP_U, ONCE>(
        z, n, tid,
        [&](const uint4v(&q)[STEP_U], int i) {
#pragma unroll
            for (int u = 0; u < STEP_U; ++u) {
                float y[N];
                unpack(q[u], y, (T*)nullptr);
                put(y, i + u * G);
            }
        },
        put);
    group_sync<G>();
    if (!unlisted.none) listed_grad<T, G>(a, out, list, 0, n, o, scale, tid);
}

// ========================================================================================================================================
// rows of few classes, at any stride: a thread per row, the classes in registers.  8 x 20 x 64^3 f32 scores with three alternatives 55 us
// = 4.8 TB/s, the gradient of 4 x 21 x 64^3 34 us = 5.2 TB/s; the distillation, whose list costs every class a comparison, is bound by its
// instructions: loss 45 us, gradient 56 us for 4 x 21 x 64^3 with four entries.
// ========================================================================================================================================
template <int CM, typename T> __device__ __forceinline__ void load_classes(float (&z)[CM], const T* p, int64_t sc, int classes) {
#pragma unroll
    for (int c = 0; c < CM; ++c) z[c] = c < classes ? to_f32(p[c * sc]) : -INFINITY;
}

template <typename T, int CM>
__global__ __launch_bounds__(256) void score_col_kernel(LogitsView v, int64_t rows, ScoreOut o) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const int classes = (int)v.classes;
    const RowPos p = row_pos(v, r);
    const T* zp = static_cast<const T*>(v.p) + row_start(v, p);
    float z[CM];
    load_classes(z, zp, v.sc, classes);
    Online on;                                                  // sums relative to the maximum itself: a row of one class scores exactly 0
    on.m = max_of(z);
    const float ref = on.m == -INFINITY ? 0.f : on.m;
#pragma unroll
    for (int c = 0; c < CM; ++c) {
        const float x = (z[c] - ref) * o.c, e = exp2_hw(x);
        on.s += e;
        on.w = fmaf(e, fmaxf(x, NEG_BIG), on.w);
    }
    const float log_s = logf(on.s);
    write_row<T, float>(o, zp, v.sc, classes, r, on.m, on.s, on.w, log_s);
    if (o.top) {
        const ListPos l = list_pos(v, p, r, o.top);
        unsigned key[CM];
#pragma unroll
        for (int c = 0; c < CM; ++c) key[c] = c < classes ? order_key(z[c]) : 0u;      // 0: taken
        for (int k = 0; k < o.top; ++k) {
            unsigned best = 0;
#pragma unroll
            for (int c = 0; c < CM; ++c) best = max(best, key[c]);
            int at = 0;
#pragma unroll
            for (int c = CM - 1; c >= 0; --c) at = key[c] == best ? c : at;             // the lowest
#pragma unroll
            for (int c = 0; c < CM; ++c) key[c] = c == at ? 0u : key[c];
            o.top_logprob[l.base + k * l.stride] = on.s != on.s ? on.s : class_logprob<float>(key_value(best), on.m, log_s, o.inv_t);
            o.top_index[l.base + k * l.stride] = at;
        }
    }
}

__device__ __forceinline__ int64_t grad_start(const LogitsView& v, RowPos p, int64_t r) { return v.class_last ? r * v.classes : p.outer * v.classes * v.inner + p.inner; }

template <typename T, int CM>
__global__ __launch_bounds__(256, 6) void score_grad_col_kernel(LogitsView v, int64_t rows, ScoreGrad o, T* __restrict__ grad) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const int classes = (int)v.classes;
    const RowPos p = row_pos(v, r);
    float z[CM];
    load_classes(z, static_cast<const T*>(v.p) + row_start(v, p), v.sc, classes);
    const float m = max_of(z), ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CM; ++c) s += exp2_hw((z[c] - ref) * o.c);
    const RowGrad g = row_grad(o, classes, r, m, s);
    T* out = grad + grad_start(v, p, r);
    const int64_t step = v.class_last ? 1 : v.inner;
#pragma unroll
    for (int c = 0; c < CM; ++c)
        if (c < classes) out[c * step] = from_f32<T>(grad_value(g, z[c]) + (c == g.token ? g.at_token : 0.f));
}

// Loss (a.loss) and / or gradient (grad) of a row; the gradient's scale: weight or the upstream gradient.  In float32, as a few classes
// leave sums of a few roundings, but for what cancels: 1 - sum p, and the loss of a good student.  The exponentials relative to the row's maximum are kept for the gradient
// (recomputed relative to the rest's maximum where the rest would underflow).  Against 64 bits its losses and gradients are
// off by 4e-7 to 9e-7 (relative, over a tensor); the row family's, whose few scalars are float64, by 6e-8.
template <typename T, int CM, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256, GRAD ? 1 : CM <= 24 ? 6 : CM <= 32 ? 5 : 1) void distill_col_kernel(LogitsView v, int64_t rows, DistillArgs a, T* __restrict__ grad) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const int classes = (int)v.classes;
    const RowPos p = row_pos(v, r);
    const ListPos l = list_pos(v, p, r, a.k);
    float z[CM], e[CM], target[CM];
    load_classes(z, static_cast<const T*>(v.p) + row_start(v, p), v.sc, classes);
    const float w = a.weight ? a.weight[r] : 1.f;
    // the teacher: tail: p = e^t, r = 1 - sum p;  else p = e^{(t - t0) - norm}
    double total = 0.0;
    float t0 = 0.f, norm = 0.f;
    if (a.tail) {
        for (int k = 0; k < a.k; ++k)
            if (load_int(a.index, l.base + k * l.stride, a.index_bytes) >= 0) total += exp((double)load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype));
    } else {
        float tmax = -INFINITY, sum = 0.f;
        for (int k = 0; k < a.k; ++k)
            if (load_int(a.index, l.base + k * l.stride, a.index_bytes) >= 0) tmax = fmaxf(tmax, load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype));
        for (int k = 0; k < a.k; ++k) {
            if (load_int(a.index, l.base + k * l.stride, a.index_bytes) < 0) continue;
            const float t = load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype);
            sum += tmax == -INFINITY ? (t != t ? t : 0.f) : exp2_hw((t - tmax) * LOG2E);
        }
        t0 = tmax == -INFINITY ? 0.f : tmax;
        norm = tmax == -INFINITY && sum != 0.f ? sum : logf(sum);
    }
    const bool nobody = !a.tail && norm == -INFINITY;                       // no entry has any probability
    const float m = max_of(z), ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CM; ++c) {
        e[c] = exp2_hw((z[c] - ref) * a.c);
        s += e[c];
        target[c] = 0.f;
    }
    const bool empty = m == -INFINITY;
    const double log_s = LOSS ? log((double)s) : (double)logf(s);
    u64 listed = 0;
    bool bad = norm != norm || total != total;
    double sum = 0.0;
    for (int k = 0; k < a.k; ++k) {
        const int64_t i = load_int(a.index, l.base + k * l.stride, a.index_bytes);
        if (i < 0) continue;
        if (i >= classes) { bad = true; continue; }
        const float lp = (load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype) - t0) - norm;
        const float pk = nobody ? 0.f : exp2_hw(lp * LOG2E);
        listed |= 1ull << i;
        float zk = 0.f;
#pragma unroll
        for (int c = 0; c < CM; ++c) {
            zk = c == (int)i ? z[c] : zk;
            target[c] += c == (int)i ? pk : 0.f;
        }
        if (LOSS && !(pk == 0.f)) sum += pk * (lp - (empty ? -INFINITY : (double)(zk - m) * a.inv_t - log_s));
    }
    float mass = nobody ? 0.f : 1.f, rest = 0.f, s_rest = 0.f;
    double log_q_rest = 0.0;
    if (a.tail) {
        float m_rest = -INFINITY;
#pragma unroll
        for (int c = 0; c < CM; ++c) {
            const bool in = (listed >> c) & 1;
            m_rest = fmaxf(m_rest, in ? -INFINITY : z[c]);
            s_rest += in ? 0.f : e[c];
        }
        double shift = 0.0;
        if (m_rest > -INFINITY && (m_rest - m) * a.c < -60.f) {             // far below the listed ones: relative to its own maximum
            shift = ((double)m_rest - m) * a.inv_t;
            s_rest = 0.f;
#pragma unroll
            for (int c = 0; c < CM; ++c) {
                if (!((listed >> c) & 1)) {
                    e[c] = exp2_hw((z[c] - m_rest) * a.c);
                    s_rest += e[c];
                }
            }
        }
        rest = s_rest > 0.f && total < 1.0 ? (float)(1.0 - total) : 0.f;
        if (!(rest > 0.f)) mass = (float)total;
        log_q_rest = shift + (LOSS ? log((double)s_rest) : (double)logf(s_rest)) - log_s;
        if (LOSS && rest > 0.f) sum += rest * (log((double)rest) - log_q_rest);
    }
    const bool nan = bad || s != s || sum != sum;
    if (LOSS) a.loss[r] = w == 0.f ? 0.f : (nan ? NAN : (float)(sum * a.t * a.t)) * w;
    if (GRAD) {
        const float scale = (a.g_loss ? a.g_loss[r] : 1.f) * w * a.t;
        const float in_f = scale * mass / s, out_f = a.tail ? (s_rest > 0.f ? scale * (mass * expf((float)log_q_rest) - rest) / s_rest : 0.f) : in_f;
        T* out = grad + grad_start(v, p, r);
        const int64_t step = v.class_last ? 1 : v.inner;
#pragma unroll
        for (int c = 0; c < CM; ++c) {
            if (c < classes) {
                const float d = (listed >> c) & 1 ? fmaf(in_f, e[c], -scale * target[c]) : out_f * e[c];
                out[c * step] = from_f32<T>(scale == 0.f ? 0.f : (nan ? NAN : (empty ? 0.f : d)));
            }
        }
    }
}

}  // namespace

// ---- launchers ---------------------------------------------------------------------------------------------------------------------------
namespace {
int vec_elems(int dtype) { return dtype == MICA_F32 ? 4 : 8; }
// Rows of up to 4096 classes take a wave each, longer ones a block: 8192 x 4000 bf16 17.4 us with a wave per row, 22.4 with a block (26.6 and
// 45.5 with five alternatives); 4096 x 16000 26.9 against 25.6.
bool wave_rows(const LogitsView& v) { return v.classes <= 4096; }
unsigned blocks_of(int64_t items, int per) { return (unsigned)((items + per - 1) / per); }

template <typename F> void by_dtype(int dtype, F&& f) {
    if (dtype == MICA_F32) f((float*)nullptr);
    else if (dtype == MICA_BF16) f((bf16_t*)nullptr);
    else f((f16_t*)nullptr);
}
template <typename F> void by_classes(int64_t c, F&& f) {
    if (c <= 8) f(std::integral_constant<int, 8>());
    else if (c <= 24) f(std::integral_constant<int, 24>());
    else if (c <= 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 64>());
}
template <typename F> void by_bool(bool b, F&& f) {
    if (b) f(std::true_type());
    else f(std::false_type());
}
}  // namespace

// f(ONCE) for a kernel that reads (READS: and nothing of the call reads the rows again) and writes (WRITES) as much as the logits hold
template <bool READS, bool WRITES, typename F> static void by_once(const LogitsView& v, int64_t rows, F&& f) {
    const int64_t size = v.dtype == MICA_F32 ? 4 : 2, bytes = rows * v.classes * size;
    const bool aligned = (((uintptr_t)v.p | (uintptr_t)(v.so * size) | (uintptr_t)(v.si * size)) & 15) == 0;
    if constexpr (READS)
        if (aligned && bytes > (int64_t)256 << 20) return f(std::integral_constant<int, ONCE_BOTH>());
    if constexpr (WRITES)
        if (bytes > (int64_t)64 << 20) return f(std::integral_constant<int, ONCE_STORE>());
    f(std::integral_constant<int, ONCE_NONE>());
}

bool score_is_col(const LogitsView& v) { return v.classes <= SCORE_COL_MAX; }

// Fewer rows than compute units, of more than 16384 classes: cut evenly so that about 256 blocks have work, into no more segments than there
// are 4096 classes begun (16385 classes: four of 3328 and one of 3073).  With
// twenty alternatives 4 x 128000 bf16 takes 11.8 us cut and 25.4 whole, 16 x 128000 12.4 and 25.6; 1 x 8000 10.7 and 7.8; without
// alternatives 64 x 128000 8.8 and 14.1, 300 x 32000 as fast whole.  And no segment beyond what a block's bits take.
SegPlan score_segments(const LogitsView& v, int64_t rows) {
    SegPlan s;
    s.n = 1;
    s.len = (int)v.classes;
    if (wave_rows(v)) return s;
    const int64_t longest = SCORE_SEG_BYTES / 16 * vec_elems(v.dtype);
    int64_t n = rows >= 256 || v.classes <= 16384 ? 1 : 256 / rows;
    n = std::min<int64_t>(n, (v.classes + 4095) / 4096);
    n = std::max<int64_t>(n, (v.classes + longest - 1) / longest);
    if (n <= 1) return s;
    int64_t len = (v.classes + n - 1) / n;
    len = (len + 63) / 64 * 64;                             // 16-byte vectors of a segment begin where the row's do; the last is not much shorter
    s.len = (int)len;
    s.n = (int)((v.classes + len - 1) / len);
    return s;
}

int64_t score_ws_bytes(const LogitsView& v, int64_t rows, int top) {
    if (score_is_col(v)) return 0;
    const SegPlan s = score_segments(v, rows);
    return s.n == 1 ? 0 : rows * s.n * ((int64_t)sizeof(Partial) + (top ? 64 * 8 : 0));
}

void launch_score(const LogitsView& v, int64_t rows, const void* tokens, int token_bytes, int64_t ignore, float temperature, int top,
                  float* logprob, float* entropy, float* lse, float* aux, float* top_logprob, int* top_index, void* ws, hipStream_t st) {
    ScoreOut o{tokens, token_bytes, ignore, logprob, entropy, lse, top_logprob, top_index, top, LOG2E / temperature, 1.0f / temperature,
               score_is_col(v) ? nullptr : aux, rows};
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        if (score_is_col(v)) {
            by_classes(v.classes, [&](auto cm) {
                hipLaunchKernelGGL((score_col_kernel<T, decltype(cm)::value>), dim3(blocks_of(rows, 256)), dim3(256), 0, st, v, rows, o);
            });
            return;
        }
        const SegPlan s = ws ? score_segments(v, rows) : SegPlan{1, (int)v.classes};      // without a workspace every row is whole
        Partial* part = static_cast<Partial*>(ws);
        u64* part_top = reinterpret_cast<u64*>(part + rows * s.n);
        const int64_t items = rows * s.n;
        by_bool(top > 0, [&](auto has_top) {
            constexpr bool TOP = decltype(has_top)::value;
            by_once<!TOP, false>(v, rows, [&](auto once) {      // the alternatives are read again
                constexpr int ONCE = decltype(once)::value;
                if (wave_rows(v)) hipLaunchKernelGGL((score_row_kernel<T, 64, TOP, ONCE>), dim3(blocks_of(items, 4)), dim3(256), 0, st, v, rows, o, s.n, s.len, part, part_top);
                else hipLaunchKernelGGL((score_row_kernel<T, 256, TOP, ONCE>), dim3((unsigned)items), dim3(256), 0, st, v, rows, o, s.n, s.len, part, part_top);
            });
            if (s.n > 1) hipLaunchKernelGGL((score_join_kernel<T, TOP>), dim3((unsigned)rows), dim3(TOP ? JOIN : 64), 0, st, v, o, s.n, part, part_top);
        });
    });
}

void launch_score_grad(const LogitsView& v, int64_t rows, const void* tokens, int token_bytes, int64_t ignore, float temperature, const float* aux,
                       const float* entropy, const float* g_logprob, const float* g_entropy, const float* g_lse, void* grad, hipStream_t st) {
    ScoreGrad o{tokens, token_bytes, ignore, aux, rows, entropy, g_logprob, g_entropy, g_lse, LOG2E / temperature, 1.0f / temperature};
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        T* out = static_cast<T*>(grad);
        if (score_is_col(v)) {
            by_classes(v.classes, [&](auto cm) {
                hipLaunchKernelGGL((score_grad_col_kernel<T, decltype(cm)::value>), dim3(blocks_of(rows, 256)), dim3(256), 0, st, v, rows, o, out);
            });
            return;
        }
        const int g = wave_rows(v) ? 64 : 256, chunk = g * UNROLL * vec_elems(v.dtype);
        const int chunks = (int)((v.classes + chunk - 1) / chunk);
        by_once<true, true>(v, rows, [&](auto once) {
            constexpr int ONCE = decltype(once)::value;
            if (g == 64) hipLaunchKernelGGL((score_grad_row_kernel<T, 64, ONCE>), dim3(blocks_of(rows * chunks, 4)), dim3(256), 0, st, v, rows, o, chunks, out);
            else hipLaunchKernelGGL((score_grad_row_kernel<T, 256, ONCE>), dim3((unsigned)(rows * chunks)), dim3(256), 0, st, v, rows, o, chunks, out);
        });
    });
}

// Threads per row in distill_step_kernel; 0: rows are too few for a block each, or a block's bits do not cover them: then in two kernels.
// 2048 / group rows are in flight on each CU, and they have to fit the 256 MB of Infinity Cache; in short rows the steps are too short for
// many waves.  us of 4096 bf16 rows, lists of 64, at 256 / 512 / 1024 threads and in two kernels:
//    32 KB   88   95  151   98       64 KB  150  152  205  175       96 KB  228  214  252  231      128 KB  297  277  301  299
//   160 KB  394  337  346  355      192 KB  492  400  402  421      250 KB  637  527  507  547
// and of rows that do not begin on 16 bytes: 65537 classes 342 317 360 360, 98305 classes 545 481 508 509.  The limits lie within 8 % of
// the best of the four on both of their sides; 500 rows differ by less (250 KB: 81 79 81 86).
static int step_group(const LogitsView& v, int64_t rows) {
    if (score_segments(v, rows).n > 1) return 0;
    if (wave_rows(v)) return 64;
    const int64_t bytes = v.classes * (v.dtype == MICA_F32 ? 4 : 2);
    return bytes <= 131072 ? 256 : bytes <= 196608 ? 512 : 1024;
}

int64_t distill_ws_bytes(const LogitsView& v, int64_t rows, bool step) {
    if (score_is_col(v)) return 0;
    const SegPlan s = score_segments(v, rows);
    return (s.n > 1 ? rows * s.n * (int64_t)sizeof(Partial) : 0) + (step && !step_group(v, rows) ? rows * 16 : 0);
}

static void distill_loss_rows(const LogitsView& v, int64_t rows, const DistillArgs& a, void* ws, hipStream_t st) {
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        const SegPlan s = score_segments(v, rows);
        Partial* part = static_cast<Partial*>(ws);
        const int64_t items = rows * s.n;
        by_bool(a.tail, [&](auto tail) {
            constexpr bool TAIL = decltype(tail)::value;
            by_once<true, false>(v, rows, [&](auto once) {
                constexpr int ONCE = decltype(once)::value;
                const auto lds = [&](int words, int groups) { return 4u * groups * (3 * a.k + (TAIL ? words : 0)); };
                if (wave_rows(v))
                    hipLaunchKernelGGL((distill_row_kernel<T, 64, TAIL, ONCE>), dim3(blocks_of(items, 4)), dim3(256), lds(mark_words<T, 64>(s.len), 4), st, v, rows, a, s.n,
                                       s.len, part);
                else
                    hipLaunchKernelGGL((distill_row_kernel<T, 256, TAIL, ONCE>), dim3((unsigned)items), dim3(256), lds(mark_words<T, 256>(s.len), 1), st, v, rows, a, s.n,
                                       s.len, part);
            });
        });
        if (s.n > 1) hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)rows), dim3(64), LIST_BYTES * a.k, st, v, rows, a, s.n, part);
    });
}
static void distill_grad_rows(const LogitsView& v, int64_t rows, const DistillArgs& a, void* grad, hipStream_t st) {
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        T* out = static_cast<T*>(grad);
        const int g = wave_rows(v) ? 64 : 256, chunk = g * UNROLL * vec_elems(v.dtype);
        const int chunks = (int)((v.classes + chunk - 1) / chunk);
        by_once<true, true>(v, rows, [&](auto once) {
            constexpr int ONCE = decltype(once)::value;
            if (g == 64) hipLaunchKernelGGL((distill_grad_row_kernel<T, 64, ONCE>), dim3(blocks_of(rows * chunks, 4)), dim3(256), 4 * LIST_BYTES * a.k, st, v, rows, a, chunks, out);
            else hipLaunchKernelGGL((distill_grad_row_kernel<T, 256, ONCE>), dim3((unsigned)(rows * chunks)), dim3(256), LIST_BYTES * a.k, st, v, rows, a, chunks, out);
        });
    });
}
template <bool LOSS, bool GRAD> static void distill_col(const LogitsView& v, int64_t rows, const DistillArgs& a, void* grad, hipStream_t st) {
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        by_classes(v.classes, [&](auto cm) {
            hipLaunchKernelGGL((distill_col_kernel<T, decltype(cm)::value, LOSS, GRAD>), dim3(blocks_of(rows, 256)), dim3(256), 0, st, v, rows, a,
                               static_cast<T*>(grad));
        });
    });
}
static DistillArgs distill_args(const DistillList& d, float temperature) {
    DistillArgs a{};
    a.index = d.index;
    a.index_bytes = d.index_bytes;
    a.teacher = d.teacher;
    a.teacher_dtype = d.teacher_dtype;
    a.k = d.k;
    a.tail = d.tail;
    a.c = LOG2E / temperature;
    a.inv_t = 1.0 / temperature;
    a.t = temperature;
    return a;
}

void launch_distill_loss(const LogitsView& v, int64_t rows, const DistillList& d, float temperature, float* loss, float* aux, void* ws, hipStream_t st) {
    DistillArgs a = distill_args(d, temperature);
    a.loss = loss;
    a.aux = aux;
    if (score_is_col(v)) distill_col<true, false>(v, rows, a, nullptr, st);
    else distill_loss_rows(v, rows, a, ws, st);
}
void launch_distill_grad(const LogitsView& v, int64_t rows, const DistillList& d, float temperature, const float* aux, const float* g_loss, void* grad,
                         hipStream_t st) {
    DistillArgs a = distill_args(d, temperature);
    a.aux = const_cast<float*>(aux);
    a.g_loss = g_loss;
    if (score_is_col(v)) distill_col<false, true>(v, rows, a, grad, st);
    else distill_grad_rows(v, rows, a, grad, st);
}
void launch_distill_step(const LogitsView& v, int64_t rows, const DistillList& d, float temperature, const float* weight, float* loss, void* grad, void* ws,
                         hipStream_t st) {
    DistillArgs a = distill_args(d, temperature);
    a.weight = weight;
    a.loss = loss;
    if (score_is_col(v)) { distill_col<true, true>(v, rows, a, grad, st); return; }
    const int group = step_group(v, rows);
    if (!group) {                                           // the row's sums first
        const SegPlan s = score_segments(v, rows);
        a.aux = reinterpret_cast<float*>(static_cast<Partial*>(ws) + (s.n > 1 ? rows * s.n : 0));
        distill_loss_rows(v, rows, a, ws, st);
        distill_grad_rows(v, rows, a, grad, st);
        return;
    }
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        T* out = static_cast<T*>(grad);
        const int n = (int)v.classes;
        by_bool(a.tail, [&](auto tail) {
            constexpr bool TAIL = decltype(tail)::value;
            by_once<false, true>(v, rows, [&](auto once) {      // the row is read again
                constexpr int ONCE = decltype(once)::value;
                const auto lds = [&](int words, int groups) { return 4u * groups * (3 * a.k + (TAIL ? words : 0)); };
                if (group == 64)
                    hipLaunchKernelGGL((distill_step_kernel<T, 64, TAIL, ONCE>), dim3(blocks_of(rows, 4)), dim3(256), lds(mark_words<T, 64, STEP_U>(n), 4), st, v, rows, a, out);
                else if (group == 256)
                    hipLaunchKernelGGL((distill_step_kernel<T, 256, TAIL, ONCE>), dim3((unsigned)rows), dim3(256), lds(mark_words<T, 256, STEP_U>(n), 1), st, v, rows, a, out);
                else if (group == 512)
                    hipLaunchKernelGGL((distill_step_kernel<T, 512, TAIL, ONCE>), dim3((unsigned)rows), dim3(512), lds(mark_words<T, 512, STEP_U>(n), 1), st, v, rows, a, out);
                else
                    hipLaunchKernelGGL((distill_step_kernel<T, 1024, TAIL, ONCE>), dim3((unsigned)rows), dim3(1024), lds(mark_words<T, 1024, STEP_U>(n), 1), st, v, rows, a, out);
            });
        });
    });
}

}  // namespace mica
