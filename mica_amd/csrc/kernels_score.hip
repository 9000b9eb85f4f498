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

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };

template <typename T> __device__ __forceinline__ uint4v load_raw(const T* p) { return *reinterpret_cast<const uint4u*>(p); }
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
template <typename T, int N> __device__ __forceinline__ void store_vec(T* p, const float (&f)[N]) {
    struct alignas(16) { T t[N]; } o;
#pragma unroll
    for (int j = 0; j < N; ++j) o.t[j] = from_f32<T>(f[j]);
    *reinterpret_cast<uint4u*>(p) = __builtin_bit_cast(uint4v, o);
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

// ---- reductions over a wave ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
template <typename F> __device__ __forceinline__ F wave_sum(F v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
template <int G> __device__ __forceinline__ void group_sync() {
    if (G == 64) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }
    else __syncthreads();
}
// over a group of G threads: a wave, or the whole block (`red`: one double per wave of the block)
template <int G> __device__ __forceinline__ float group_max(float v, double* red) {
    v = wave_max(v);
    if (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (float)red[0];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) v = fmaxf(v, (float)red[i]);
    }
    return v;
}
template <int G> __device__ __forceinline__ double group_sum(double v, double* red) {
    v = wave_sum(v);
    if (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) v += red[i];
    }
    return v;
}

// ---- the 64 largest keys of a wave: one per lane, descending ------------------------------------------------------------------------
__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) {
    const unsigned lo = __shfl_xor((unsigned)v, o), hi = __shfl_xor((unsigned)(v >> 32), o);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 shfl64(u64 v, int l) {
    const unsigned lo = __shfl((unsigned)v, l), hi = __shfl((unsigned)(v >> 32), l);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 cmp_exchange(u64 v, int o, bool take_max) {
    const u64 w = shfl_xor64(v, o);
    return (v > w) == take_max ? v : w;
}
__device__ __forceinline__ u64 bitonic_merge64(u64 v, int lane) {      // a bitonic sequence -> descending
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = cmp_exchange(v, o, (lane & o) == 0);
    return v;
}
__device__ __forceinline__ u64 sort64(u64 v, int lane) {               // descending
#pragma unroll
    for (int k = 2; k < 64; k <<= 1)
#pragma unroll
        for (int o = k >> 1; o > 0; o >>= 1) v = cmp_exchange(v, o, ((lane & o) == 0) == ((lane & k) == 0));
    return bitonic_merge64(v, lane);
}
// a, b descending, b given reversed (lane i holds the (63 - i)-th): the 64 largest of both, descending
__device__ __forceinline__ u64 merge_top64(u64 a, u64 b_reversed, int lane) { return bitonic_merge64(a > b_reversed ? a : b_reversed, lane); }

// ---- online softmax of one thread -----------------------------------------------------------------------------------------------------
// m: running maximum, s = sum 2^{(z - m) c}, w = sum 2^{(z - m) c} (z - m) c.  Differences to the maximum, not z c - m c: a row of the
// type's lowest values would overflow there.
struct Online {
    float m = -INFINITY, s = 0.f, w = 0.f;
    template <int N, bool ENT> __device__ __forceinline__ void add(const float (&f)[N], float vmax, float c) {
        const float mn = fmaxf(m, vmax);
        const float d = fmaxf((m - mn) * c, NEG_BIG);         // -inf - -inf = NaN -> NEG_BIG, with s = w = 0
        const float a = exp2_hw(d);
        if (ENT) w = a * fmaf(s, d, w);
        s *= a;
        m = mn;
        const float ref = mn == -INFINITY ? 0.f : mn;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float x = (f[j] - ref) * c;
            const float e = exp2_hw(x);
            s += e;
            if (ENT) w = fmaf(e, fmaxf(x, NEG_BIG), w);
        }
    }
    // rescaled to a maximum >= m
    __device__ __forceinline__ void rescale(float mn, float c) {
        const float d = fmaxf((m - mn) * c, NEG_BIG);
        const float a = m == -INFINITY ? 0.f : exp2_hw(d);
        w = m == -INFINITY && s == 0.f ? 0.f : a * fmaf(s, d, w);
        s = m == -INFINITY && s == 0.f ? 0.f : (m == -INFINITY ? s : s * a);      // a NaN row keeps its NaN
        m = mn;
    }
};

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

// Streams the n classes at z: f(values[N], first index) for every 16-byte vector of this thread, values beyond n = -inf.
template <typename T, int G, typename F> __device__ __forceinline__ void stream_row(const T* __restrict__ z, int n, int tid, F&& f) {
    constexpr int N = Vec<T>::N;
    const int nfull = n / N;
    int i = tid;
    for (; i + (UNROLL - 1) * G < nfull; i += UNROLL * G) {
        uint4v q[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) q[u] = load_raw(z + (int64_t)(i + u * G) * N);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[N];
            unpack(q[u], v, (T*)nullptr);
            f(v, (i + u * G) * N);
        }
    }
    for (; i < nfull; i += G) {
        float v[N];
        unpack(load_raw(z + (int64_t)i * N), v, (T*)nullptr);
        f(v, i * N);
    }
    if (i == nfull && nfull * N < n) {
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = nfull * N + j < n ? to_f32(z[nfull * N + j]) : -INFINITY;
        f(v, nfull * N);
    }
}

// The K <= 64 largest of a group's row.  While streaming, every thread notes its largest value and the vector that held it first.  The
// K-th largest of these (value, position) pairs bounds the K-th largest element from below, so only the threads at or above the bound
// can own one of the K: their vectors are read once more (K / G of the row, from cache) and what passes the bound is merged, 64 keys at
// a time, into a sorted list that each wave holds one key per lane.  Exact for any data; ties and -inf order by index.
struct TopScratch {             // LDS of one wave
    u64 list[64];
    u64 buf[128];
};
template <typename T, int G>
__device__ __forceinline__ u64 group_top(const T* __restrict__ z, int n, unsigned index0, int k, float best, int best_at, bool any, TopScratch* sc,
                                         int* owners, int* nown) {
    constexpr int N = Vec<T>::N, NW = G / 64;
    const int tid = G == 64 ? (threadIdx.x & 63) : threadIdx.x, lane = threadIdx.x & 63, w = G == 64 ? 0 : threadIdx.x >> 6;
    const u64 mine = any ? make_key(order_key(best), (unsigned)best_at) : 0;
    u64 sorted = sort64(mine, lane);
    if (NW > 1) {
        sc[w].list[lane] = sorted;
        if (threadIdx.x == 0) *nown = 0;
        __syncthreads();
        sorted = sc[0].list[lane];
#pragma unroll
        for (int i = 1; i < NW; ++i) sorted = merge_top64(sorted, sc[i].list[63 - lane], lane);
    }
    const u64 bound = shfl64(sorted, k - 1);
    int count;
    if (NW > 1) {
        const bool own = any && mine >= bound;
        if (own) owners[atomicAdd(nown, 1)] = tid;      // the order of the owners does not change the result
        __syncthreads();
        count = *nown;
    } else {
        const u64 b = __ballot(any && mine >= bound);
        if (any && mine >= bound) owners[__popcll(b & ((1ull << lane) - 1))] = tid;
        wave_sync();
        count = __popcll(b);
    }
    const int nvec = (n + N - 1) / N, per = (nvec + G - 1) / G;
    const int64_t total = (int64_t)count * per;
    u64 list = 0, floor_key = 0;
    int pending = 0;
    for (int64_t p0 = 0; p0 < total; p0 += G) {
        const int64_t p = p0 + tid;
        const int vec = p < total ? owners[p % count] + (int)(p / count) * G : nvec;
        float v[N];
        if ((vec + 1) * N <= n) unpack(load_raw(z + (int64_t)vec * N), v, (T*)nullptr);
        else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = vec * N + j < n ? to_f32(z[vec * N + j]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = vec * N + j;
            const unsigned o = order_key(v[j]);
            const u64 key = make_key(o, (unsigned)at);
            const bool pass = at < n && make_key(o, (unsigned)(vec * N)) >= bound && key > floor_key;
            const u64 b = __ballot(pass);
            if (b == 0) continue;
            if (pass) sc[w].buf[pending + __popcll(b & ((1ull << lane) - 1))] = key;
            pending += __popcll(b);
            wave_sync();
            if (pending >= 64) {
                const u64 take = sc[w].buf[lane], rest = sc[w].buf[64 + lane];
                wave_sync();
                sc[w].buf[lane] = rest;
                wave_sync();
                pending -= 64;
                const u64 s = sort64(take, lane);
                list = merge_top64(list, shfl64(s, 63 - lane), lane);
                floor_key = shfl64(list, k - 1);
            }
        }
    }
    if (pending > 0) {
        const u64 s = sort64(lane < pending ? sc[w].buf[lane] : 0, lane);
        list = merge_top64(list, shfl64(s, 63 - lane), lane);
    }
    if (NW > 1) {
        __syncthreads();
        sc[w].list[lane] = list;
        __syncthreads();
        list = sc[0].list[lane];
#pragma unroll
        for (int i = 1; i < NW; ++i) list = merge_top64(list, sc[i].list[63 - lane], lane);
    }
    // classes are numbered within the segment so far
    return list == 0 ? 0 : ((list & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (key_index(list) + index0)));
}

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
};
// natural logarithm of the sum relative to the maximum
__device__ __forceinline__ float row_lse(float m, float log_s, float inv_t) { return m == -INFINITY ? -INFINITY : (float)((double)m * inv_t + log_s); }
__device__ __forceinline__ float class_logprob(float z, float m, float log_s, float inv_t) {
    return m == -INFINITY ? (log_s != log_s ? log_s : -INFINITY) : (float)((double)(z - m) * inv_t - log_s);
}
template <typename T>
__device__ __forceinline__ void write_row(const ScoreOut& o, const T* __restrict__ z, int64_t sc, int64_t classes, int64_t r, float m, float s, float w) {
    const float log_s = (float)log((double)s);            // s >= 1 unless the row is empty (0) or holds NaN
    o.lse[r] = s != s ? s : row_lse(m, log_s, o.inv_t);
    o.entropy[r] = s == 0.f ? 0.f : (float)(LN2 * (log2((double)s) - (double)w / s));
    if (o.logprob) {
        const int64_t t = load_int(o.tokens, r, o.token_bytes);
        float lp;
        if (t == o.ignore) lp = 0.f;
        else if (t < 0 || t >= classes) lp = NAN;
        else lp = s != s ? s : class_logprob(to_f32(z[t * sc]), m, log_s, o.inv_t);
        o.logprob[r] = lp;
    }
}
__device__ __forceinline__ void write_top(const ScoreOut& o, const LogitsView& v, RowPos p, int64_t r, u64 key, int lane, float m, float s) {
    if (lane < o.top) {
        const float log_s = (float)log((double)s);
        const ListPos l = list_pos(v, p, r, o.top);
        o.top_logprob[l.base + lane * l.stride] = s != s ? s : class_logprob(key_value((unsigned)(key >> 32)), m, log_s, o.inv_t);
        o.top_index[l.base + lane * l.stride] = (int)key_index(key);
    }
}

struct Partial { float m, s, w, unused; };                 // of one segment of a row

template <typename T, int G, bool TOP>
__global__ __launch_bounds__(256) void score_row_kernel(LogitsView v, int64_t rows, ScoreOut o, int segments, int seg_len, Partial* __restrict__ part,
                                                        u64* __restrict__ part_top) {
    constexpr int NW = G / 64, GROUPS = 256 / G;
    __shared__ double red[4];
    __shared__ TopScratch top_sc[TOP ? 4 : 1];
    __shared__ int owners[TOP ? 256 : 1];
    __shared__ int nown;
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
    float best = -INFINITY;
    int best_at = 0;
    bool any = false;
    stream_row<T, G>(z + first, n, tid, [&](const float(&f)[Vec<T>::N], int at) {
        const float vm = max_of(f);
        if (TOP) {
            if (!any || vm > best) { best = vm; best_at = at; }
            any = true;
        }
        on.add<Vec<T>::N, true>(f, vm, o.c);
    });
    const float m = group_max<G>(on.m, red);
    on.rescale(m, o.c);
    const float s = (float)group_sum<G>((double)on.s, red), w = (float)group_sum<G>((double)on.w, red);
    u64 key = 0;
    if (TOP) key = group_top<T, G>(z + first, n, (unsigned)first, o.top, best, best_at, any, NW == 1 ? &top_sc[g] : top_sc, &owners[g * G], &nown);
    if (segments == 1) {
        if (tid == 0) write_row<T>(o, z, 1, v.classes, r, m, s, w);
        if (TOP && tid < 64) write_top(o, v, p, r, key, lane, m, s);
    } else {
        if (tid == 0) part[item] = {m, s, w, 0.f};
        if (TOP && tid < o.top) part_top[item * 64 + tid] = key;
    }
}

// joins the segments of a row: one block of 256
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void score_join_kernel(LogitsView v, ScoreOut o, int segments, const Partial* __restrict__ part,
                                                         const u64* __restrict__ part_top) {
    __shared__ double red[4];
    __shared__ u64 lists[4][64];
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    Online on;
    for (int i = threadIdx.x; i < segments; i += 256) {
        const Partial q = part[r * segments + i];
        Online b;
        b.m = q.m; b.s = q.s; b.w = q.w;
        const float mn = fmaxf(on.m, q.m);
        on.rescale(mn, o.c);
        b.rescale(mn, o.c);
        on.s += b.s;
        on.w += b.w;
    }
    const float m = group_max<256>(on.m, red);
    on.rescale(m, o.c);
    const float s = (float)group_sum<256>((double)on.s, red), ws = (float)group_sum<256>((double)on.w, red);
    if (threadIdx.x == 0) write_row<T>(o, z, 1, v.classes, r, m, s, ws);
    if (TOP) {
        u64 list = 0;
        for (int i = w; i < segments; i += 4) {
            const u64* q = part_top + (r * segments + i) * 64;
            list = merge_top64(list, 63 - lane < o.top ? q[63 - lane] : 0, lane);
        }
        lists[w][lane] = list;
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int i = 1; i < 4; ++i) list = merge_top64(list, lists[i][63 - lane], lane);
            write_top(o, v, p, r, list, lane, m, s);
        }
    }
}

// ---- gradient of the scores ------------------------------------------------------------------------------------------------------------
// dz_v = (1/T) [ g_lp ([v = t] - p_v) + g_lse p_v - g_H p_v (log p_v + H) ]: one read, one write, no state but lse and H
struct ScoreGrad {
    const void* tokens;
    int token_bytes;
    int64_t ignore;
    const float* lse;
    const float* entropy;
    const float* g_logprob;
    const float* g_entropy;
    const float* g_lse;
    float c, inv_t;
};
struct RowGrad {
    float l2;           // lse in units of log 2
    float a;            // coefficient of p
    float b;            // coefficient of p log2 p
    float at_token;     // added at the token
    int64_t token;      // -1: none
    bool empty;
};
__device__ __forceinline__ RowGrad row_grad(const ScoreGrad& o, int64_t classes, int64_t r) {
    RowGrad g;
    const float lse = o.lse[r];
    g.empty = lse == -INFINITY;
    g.l2 = lse * LOG2E;
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
    g.a = (gl - glp - (ge != 0.f ? ge * o.entropy[r] : 0.f)) * o.inv_t;
    g.b = -ge * (float)LN2 * o.inv_t;
    g.at_token = g.empty ? 0.f : glp * o.inv_t;
    return g;
}
__device__ __forceinline__ float grad_value(const RowGrad& g, float z, float c) {
    const float x = fmaf(z, c, -g.l2);
    const float p = exp2_hw(x);
    return g.empty ? 0.f : p * fmaf(g.b, fmaxf(x, NEG_BIG), g.a);
}

// what a block of the gradient kernels covers: G threads x UNROLL vectors of one row
template <typename T, int G, typename F>
__device__ __forceinline__ void map_chunk(const T* __restrict__ z, T* __restrict__ out, int first, int64_t classes, int tid, F&& f) {
    constexpr int N = Vec<T>::N;
    uint4v q[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t at = first + (int64_t)(tid + u * G) * N;
        if (at + N <= classes) q[u] = load_raw(z + at);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t at = first + (int64_t)(tid + u * G) * N;
        if (at + N <= classes) {
            float v[N];
            unpack(q[u], v, (T*)nullptr);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = f(v[j], at + j);
            store_vec(out + at, v);
        } else {
            for (int j = 0; j < N; ++j)
                if (at + j < classes) out[at + j] = from_f32<T>(f(to_f32(z[at + j]), at + j));
        }
    }
}

template <typename T, int G>
__global__ __launch_bounds__(256) void score_grad_row_kernel(LogitsView v, int64_t rows, ScoreGrad o, int chunks, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / G, CHUNK = G * UNROLL * Vec<T>::N;
    const int tid = threadIdx.x % G;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G;
    if (item >= rows * chunks) return;
    const int64_t r = chunks == 1 ? item : item / chunks;
    const int first = chunks == 1 ? 0 : (int)(item % chunks) * CHUNK;
    const RowGrad g = row_grad(o, v.classes, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, row_pos(v, r));
    map_chunk<T, G>(z, grad + r * v.classes, first, v.classes, tid,
                    [&](float x, int64_t at) { return grad_value(g, x, o.c) + (at == g.token ? g.at_token : 0.f); });
}

// ---- distillation ------------------------------------------------------------------------------------------------------------------------
struct DistillArgs {
    const void* index;
    int index_bytes;
    const void* teacher;
    int teacher_dtype;
    int k;
    int tail;
    float c, inv_t, t;
    const float* weight;          // nullable: rows of weight 0 are skipped
    float* loss;
    float* aux;                   // [4][rows], nullable: ref, factor, lse, mass (tail) or the teacher's log sum
    const float* g_loss;          // gradient kernels
};
// A row's gradient: factor * e^{y - ref} where a class is not listed, mass * e^{y - lse} - sum p at a listed one, times T and the
// upstream gradient.  (tail: ref is the log sum of the classes that are not listed and factor = mass q_rest - r, so that nothing
// overflows where q_rest is tiny; else ref = lse, factor = mass.)
struct RowDistill { float loss, ref, factor, lse, mass, norm; bool skip; };

// dynamic LDS of a distill group: K indices, then a bit per class of the segment (tail)
template <typename T, int G>
__device__ __forceinline__ bool list_load(const DistillArgs& a, ListPos l, int tid, int* idx) {
    bool used = false;
    for (int k = tid; k < a.k; k += G) {
        const int64_t i = load_int(a.index, l.base + k * l.stride, a.index_bytes);
        idx[k] = i < 0 ? -1 : (i > 0x7FFFFFFE ? 0x7FFFFFFF : (int)i);
        used |= i >= 0;
    }
    return used;
}
template <int G> __device__ __forceinline__ void mark_listed(const int* idx, int k, int first, int n, unsigned* bits, int tid) {
    for (int i = tid; i < (n + 31) / 32; i += G) bits[i] = 0;
    group_sync<G>();
    for (int i = tid; i < k; i += G) {
        const int v = idx[i] - first;
        if (idx[i] >= 0 && v >= 0 && v < n) atomicOr(&bits[v >> 5], 1u << (v & 31));
    }
    group_sync<G>();
}
// the online sums of the classes of a segment, without the listed ones if TAIL
template <typename T, int G, bool TAIL>
__device__ __forceinline__ Online distill_stream(const T* __restrict__ z, int n, int tid, const unsigned* bits, float c) {
    constexpr int N = Vec<T>::N;
    Online on;
    stream_row<T, G>(z, n, tid, [&](const float(&f0)[N], int at) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = f0[j];
        if (TAIL) {
            const unsigned b = (bits[at >> 5] >> (at & 31)) & ((1u << N) - 1u);
            if (b) {
#pragma unroll
                for (int j = 0; j < N; ++j) f[j] = (b >> j) & 1u ? -INFINITY : f[j];
            }
        }
        on.add<N, false>(f, max_of(f), c);
    });
    return on;
}

// The row's loss and what its gradient needs, from the sums (m, s) over all classes, or over the classes that are not listed (tail).
// All threads of the group; idx in LDS.
template <typename T, int G>
__device__ __forceinline__ RowDistill distill_finish(const DistillArgs& a, const T* __restrict__ z, int64_t classes, ListPos l, const int* idx,
                                                     float m, float s, int tid, double* red) {
    RowDistill o;
    o.skip = false;
    bool bad = false;
    float tmax = -INFINITY, zmax = -INFINITY;
    for (int k = tid; k < a.k; k += G) {
        const int i = idx[k];
        if (i < 0) continue;
        if (i >= classes) { bad = true; continue; }
        tmax = fmaxf(tmax, load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype));
        zmax = fmaxf(zmax, to_f32(z[i]));
    }
    zmax = group_max<G>(zmax, red);
    double norm = 0.0, mass = 1.0, rest = 0.0, log_q_rest = 0.0, lse, lse_rest = 0.0;
    double M = m, log_s;                                        // maximum and log sum of all classes
    if (!a.tail) {
        tmax = group_max<G>(tmax, red);
        double e = 0.0;
        for (int k = tid; k < a.k; k += G) {
            const int i = idx[k];
            if (i >= 0 && i < classes) {
                const float t = load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype);
                e += tmax == -INFINITY ? (t != t ? (double)t : 0.0) : exp((double)t - tmax);
            }
        }
        e = group_sum<G>(e, red);
        norm = e == 0.0 ? -INFINITY : (tmax == -INFINITY ? e : tmax + log(e));
        mass = e == 0.0 ? 0.0 : 1.0;
        log_s = log((double)s);
    } else {
        double sl = 0.0, P = 0.0;
        for (int k = tid; k < a.k; k += G) {
            const int i = idx[k];
            if (i < 0 || i >= classes) continue;
            P += exp((double)load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype));
            bool again = false;
            for (int j = 0; j < k; ++j) again |= idx[j] == i;
            const float zk = to_f32(z[i]);
            if (!again) sl += zmax == -INFINITY ? (zk != zk ? (double)zk : 0.0) : (double)exp2_hw((zk - zmax) * a.c);
        }
        sl = group_sum<G>(sl, red);
        P = group_sum<G>(P, red);
        const bool have_rest = !(s == 0.f);                      // NaN counts
        rest = have_rest ? (P < 1.0 ? 1.0 - P : 0.0) : 0.0;
        mass = P + rest;
        if (!have_rest) { M = zmax; log_s = log(sl); }
        else if (sl == 0.0) { log_s = log((double)s); lse_rest = (double)m * a.inv_t + log_s; }
        else {
            M = fmaxf(m, zmax);
            const double u = ((double)zmax - m) * a.inv_t + log(sl) - log((double)s);      // log of (listed sum / rest sum)
            log_q_rest = -(u > 700.0 ? u : log1p(exp(u)));
            lse_rest = (double)m * a.inv_t + log((double)s);
            log_s = lse_rest - log_q_rest - M * a.inv_t;
        }
    }
    lse = M == -INFINITY ? -INFINITY : M * a.inv_t + log_s;
    double sum = 0.0;
    for (int k = tid; k < a.k; k += G) {
        const int i = idx[k];
        if (i < 0 || i >= classes) continue;
        const double lp = (double)load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype) - norm;
        const double pk = mass == 0.0 ? 0.0 : exp(lp);
        const double lq = lse == -INFINITY ? -INFINITY : ((double)to_f32(z[i]) - M) * a.inv_t - log_s;
        if (!(pk == 0.0)) sum += pk * (lp - lq);
    }
    if (bad) sum = NAN;
    sum = group_sum<G>(sum, red);
    if (rest > 0.0) sum += rest * (log(rest) - log_q_rest);
    const bool nan_row = s != s;
    o.loss = nan_row ? NAN : (float)(sum * a.t * a.t);
    o.lse = nan_row ? NAN : (float)lse;
    o.mass = (float)mass;
    o.norm = (float)norm;
    if (a.tail) {
        const bool have_rest = !(s == 0.f);
        o.ref = have_rest ? (float)lse_rest : 0.f;
        o.factor = have_rest ? (float)(mass * exp(log_q_rest) - rest) : 0.f;
    } else {
        o.ref = o.lse;
        o.factor = o.mass;
    }
    if (sum != sum) o.factor = NAN;                              // an invalid entry shows in the gradient too
    return o;
}

template <typename T, int G, bool TAIL>
__global__ __launch_bounds__(256) void distill_row_kernel(LogitsView v, int64_t rows, DistillArgs a, int segments, int seg_len, Partial* __restrict__ part) {
    constexpr int GROUPS = 256 / G;
    extern __shared__ int dyn[];
    __shared__ double red[4];
    const int g = threadIdx.x / G, tid = threadIdx.x % G;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + g;
    if (item >= rows * segments) return;
    const int64_t r = segments == 1 ? item : item / segments;
    const int seg = segments == 1 ? 0 : (int)(item % segments);
    const int words = TAIL ? (seg_len + 31) / 32 : 0;
    int* idx = dyn + g * (a.k + words);
    unsigned* bits = reinterpret_cast<unsigned*>(idx + a.k);
    const RowPos p = row_pos(v, r);
    const ListPos l = list_pos(v, p, r, a.k);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    const int first = seg * seg_len;
    const int n = (int)(v.classes - first < seg_len ? v.classes - first : seg_len);
    list_load<T, G>(a, l, tid, idx);
    group_sync<G>();
    if (TAIL) mark_listed<G>(idx, a.k, first, n, bits, tid);
    Online on = distill_stream<T, G, TAIL>(z + first, n, tid, bits, a.c);
    const float m = group_max<G>(on.m, red);
    on.rescale(m, a.c);
    const float s = (float)group_sum<G>((double)on.s, red);
    if (segments > 1) {
        if (tid == 0) part[item] = {m, s, 0.f, 0.f};
        return;
    }
    const RowDistill o = distill_finish<T, G>(a, z, v.classes, l, idx, m, s, tid, red);
    if (tid == 0) {
        const float w = a.weight ? a.weight[r] : 1.f;
        a.loss[r] = w == 0.f ? 0.f : o.loss * w;
        if (a.aux) {
            a.aux[r] = o.ref;
            a.aux[rows + r] = o.factor;
            a.aux[2 * rows + r] = o.lse;
            a.aux[3 * rows + r] = a.tail ? o.mass : o.norm;
        }
    }
}
template <typename T>
__global__ __launch_bounds__(256) void distill_join_kernel(LogitsView v, int64_t rows, DistillArgs a, int segments, const Partial* __restrict__ part) {
    extern __shared__ int dyn[];
    __shared__ double red[4];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const RowPos p = row_pos(v, r);
    const ListPos l = list_pos(v, p, r, a.k);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    list_load<T, 256>(a, l, tid, dyn);
    Online on;
    for (int i = tid; i < segments; i += 256) {
        const Partial q = part[r * segments + i];
        Online b;
        b.m = q.m; b.s = q.s;
        const float mn = fmaxf(on.m, q.m);
        on.rescale(mn, a.c);
        b.rescale(mn, a.c);
        on.s += b.s;
    }
    const float m = group_max<256>(on.m, red);
    on.rescale(m, a.c);
    const float s = (float)group_sum<256>((double)on.s, red);
    const RowDistill o = distill_finish<T, 256>(a, z, v.classes, l, dyn, m, s, tid, red);
    if (tid == 0) {
        const float w = a.weight ? a.weight[r] : 1.f;
        a.loss[r] = w == 0.f ? 0.f : o.loss * w;
        if (a.aux) {
            a.aux[r] = o.ref;
            a.aux[rows + r] = o.factor;
            a.aux[2 * rows + r] = o.lse;
            a.aux[3 * rows + r] = a.tail ? o.mass : o.norm;
        }
    }
}

// the listed classes of [first, first + n): overwrites what the sweep wrote there; the first mention of a class writes for all of them
template <typename T, int G>
__device__ __forceinline__ void listed_grad(const DistillArgs& a, const T* __restrict__ z, T* __restrict__ out, int64_t classes, ListPos l, const int* idx,
                                            int64_t first, int64_t n, float lse, float mass, float norm, float scale, int tid) {
    for (int k = tid; k < a.k; k += G) {
        const int i = idx[k];
        if (i < 0 || i >= classes || i < first || i >= first + n) continue;
        bool again = false;
        for (int j = 0; j < k; ++j) again |= idx[j] == i;
        if (again) continue;
        float p = 0.f;
        for (int j = k; j < a.k; ++j)
            if (idx[j] == i) {
                const float t = load_float(a.teacher, l.base + j * l.stride, a.teacher_dtype);
                p += a.tail ? expf(t) : (norm == -INFINITY ? 0.f : expf(t - norm));
            }
        const float q = lse == -INFINITY ? 0.f : exp2_hw(fmaf(to_f32(z[i]), a.c, -lse * LOG2E));
        out[i] = from_f32<T>(lse == -INFINITY ? 0.f : scale * (mass * q - p));
    }
}
__device__ __forceinline__ float unlisted_grad(float z, float ref2, float f, float c) { return f * exp2_hw(fmaf(z, c, -ref2)); }

template <typename T, int G>
__global__ __launch_bounds__(256) void distill_grad_row_kernel(LogitsView v, int64_t rows, DistillArgs a, int chunks, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / G, CHUNK = G * UNROLL * Vec<T>::N;
    extern __shared__ int dyn[];
    const int g = threadIdx.x / G, tid = threadIdx.x % G;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + g;
    if (item >= rows * chunks) return;
    const int64_t r = chunks == 1 ? item : item / chunks;
    const int first = chunks == 1 ? 0 : (int)(item % chunks) * CHUNK;
    int* idx = dyn + g * a.k;
    const RowPos p = row_pos(v, r);
    const ListPos l = list_pos(v, p, r, a.k);
    list_load<T, G>(a, l, tid, idx);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    T* out = grad + r * v.classes;
    const float up = (a.g_loss ? a.g_loss[r] : 1.f) * (a.weight ? a.weight[r] : 1.f);
    const float scale = up * a.t;
    const float ref = a.aux[r], factor = a.aux[rows + r], lse = a.aux[2 * rows + r], x = a.aux[3 * rows + r];
    const float mass = a.tail ? x : (x == -INFINITY ? 0.f : 1.f), norm = a.tail ? 0.f : x;
    const bool none = lse == -INFINITY || (a.weight && a.weight[r] == 0.f);
    const float ref2 = none ? 0.f : ref * LOG2E, f = scale * factor;
    map_chunk<T, G>(z, out, first, v.classes, tid, [&](float y, int64_t) { return none ? 0.f : unlisted_grad(y, ref2, f, a.c); });
    group_sync<G>();
    if (!none) listed_grad<T, G>(a, z, out, v.classes, l, idx, first, CHUNK, lse, mass, norm, scale, tid);
}

// loss and gradient in one kernel: the row is read twice, the second time from cache, and its gradient written
template <typename T, int G, bool TAIL>
__global__ __launch_bounds__(256) void distill_step_row_kernel(LogitsView v, int64_t rows, DistillArgs a, T* __restrict__ grad) {
    constexpr int GROUPS = 256 / G, N = Vec<T>::N;
    extern __shared__ int dyn[];
    __shared__ double red[4];
    const int g = threadIdx.x / G, tid = threadIdx.x % G;
    const int64_t r = (int64_t)blockIdx.x * GROUPS + g;
    if (r >= rows) return;
    const int words = TAIL ? (int)((v.classes + 31) / 32) : 0;
    int* idx = dyn + g * (a.k + words);
    unsigned* bits = reinterpret_cast<unsigned*>(idx + a.k);
    const RowPos p = row_pos(v, r);
    const ListPos l = list_pos(v, p, r, a.k);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    T* out = grad + r * v.classes;
    const float w = a.weight ? a.weight[r] : 1.f;
    list_load<T, G>(a, l, tid, idx);
    group_sync<G>();
    if (TAIL) mark_listed<G>(idx, a.k, 0, (int)v.classes, bits, tid);
    Online on = distill_stream<T, G, TAIL>(z, (int)v.classes, tid, bits, a.c);
    const float m = group_max<G>(on.m, red);
    on.rescale(m, a.c);
    const float s = (float)group_sum<G>((double)on.s, red);
    const RowDistill o = distill_finish<T, G>(a, z, v.classes, l, idx, m, s, tid, red);
    if (tid == 0) a.loss[r] = w == 0.f ? 0.f : o.loss * w;
    const float scale = w * a.t;
    const bool none = o.lse == -INFINITY || w == 0.f;
    const float ref2 = none ? 0.f : o.ref * LOG2E, f = scale * o.factor;
    stream_row<T, G>(z, (int)v.classes, tid, [&](const float(&y)[N], int at) {
        float d[N];
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] = none ? 0.f : unlisted_grad(y[j], ref2, f, a.c);
        if (at + N <= v.classes) store_vec(out + at, d);
        else {
            for (int j = 0; j < N; ++j)
                if (at + j < v.classes) out[at + j] = from_f32<T>(d[j]);
        }
    });
    group_sync<G>();
    if (!none) listed_grad<T, G>(a, z, out, v.classes, l, idx, 0, v.classes, o.lse, o.mass, o.norm, scale, tid);
}

// ========================================================================================================================================
// rows of few classes, at any stride: a thread per row, the classes in registers
// ========================================================================================================================================
template <int CM> struct ColRow {
    float z[CM];
    float m, s;
    template <typename T> __device__ __forceinline__ void load(const T* p, int64_t sc, int classes) {
#pragma unroll
        for (int c = 0; c < CM; ++c) z[c] = c < classes ? to_f32(p[c * sc]) : -INFINITY;
    }
};

template <typename T, int CM>
__global__ __launch_bounds__(256) void score_col_kernel(LogitsView v, int64_t rows, ScoreOut o) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const int classes = (int)v.classes;
    const RowPos p = row_pos(v, r);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    ColRow<CM> x;
    x.load(z, v.sc, classes);
    Online on;
    on.add<CM, true>(x.z, max_of(x.z), o.c);
    write_row<T>(o, z, v.sc, classes, r, on.m, on.s, on.w);
    if (o.top) {
        const float log_s = (float)log((double)on.s);
        const ListPos l = list_pos(v, p, r, o.top);
        u64 last = ~0ull;
        for (int k = 0; k < o.top; ++k) {                      // the largest key below the last one
            u64 best = 0;
#pragma unroll
            for (int c = 0; c < CM; ++c) {
                const u64 key = make_key(order_key(x.z[c]), c);
                if (c < classes && key < last && key > best) best = key;
            }
            last = best;
            o.top_logprob[l.base + k * l.stride] = on.s != on.s ? on.s : class_logprob(key_value((unsigned)(best >> 32)), on.m, log_s, o.inv_t);
            o.top_index[l.base + k * l.stride] = (int)key_index(best);
        }
    }
}

__device__ __forceinline__ int64_t grad_start(const LogitsView& v, RowPos p, int64_t r) { return v.class_last ? r * v.classes : p.outer * v.classes * v.inner + p.inner; }

template <typename T, int CM>
__global__ __launch_bounds__(256) void score_grad_col_kernel(LogitsView v, int64_t rows, ScoreGrad o, T* __restrict__ grad) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const int classes = (int)v.classes;
    const RowPos p = row_pos(v, r);
    ColRow<CM> x;
    x.load(static_cast<const T*>(v.p) + row_start(v, p), v.sc, classes);
    const RowGrad g = row_grad(o, classes, r);
    T* out = grad + grad_start(v, p, r);
    const int64_t step = v.class_last ? 1 : v.inner;
#pragma unroll
    for (int c = 0; c < CM; ++c)
        if (c < classes) out[c * step] = from_f32<T>(grad_value(g, x.z[c], o.c) + (c == g.token ? g.at_token : 0.f));
}

// loss (a.loss) and / or gradient (grad) of a row; the gradient's scale: weight or the upstream gradient
template <typename T, int CM, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256) void distill_col_kernel(LogitsView v, int64_t rows, DistillArgs a, T* __restrict__ grad) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const int classes = (int)v.classes;
    const RowPos p = row_pos(v, r);
    const ListPos l = list_pos(v, p, r, a.k);
    const T* z = static_cast<const T*>(v.p) + row_start(v, p);
    ColRow<CM> x;
    x.load(z, v.sc, classes);
    const float w = a.weight ? a.weight[r] : 1.f;
    // the teacher's probability of each class
    float target[CM];
#pragma unroll
    for (int c = 0; c < CM; ++c) target[c] = 0.f;
    u64 listed = 0;
    bool bad = false;
    float tmax = -INFINITY;
    double norm = 0.0, P = 0.0;
    if (!a.tail) {
        for (int k = 0; k < a.k; ++k) {
            const int64_t i = load_int(a.index, l.base + k * l.stride, a.index_bytes);
            if (i >= 0) tmax = fmaxf(tmax, load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype));
        }
        double e = 0.0;
        for (int k = 0; k < a.k; ++k) {
            const int64_t i = load_int(a.index, l.base + k * l.stride, a.index_bytes);
            const float t = load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype);
            if (i >= 0) e += tmax == -INFINITY ? (t != t ? (double)t : 0.0) : exp((double)t - tmax);
        }
        norm = e == 0.0 ? -INFINITY : (tmax == -INFINITY ? e : tmax + log(e));
    }
    const float m_all = max_of(x.z);
    Online on;
    on.add<CM, false>(x.z, m_all, a.c);
    const bool empty = on.s == 0.f;
    const double log_all = log((double)on.s);
    double sum = 0.0;
    for (int k = 0; k < a.k; ++k) {
        const int64_t i = load_int(a.index, l.base + k * l.stride, a.index_bytes);
        if (i < 0) continue;
        if (i >= classes) { bad = true; continue; }
        const double lp = (double)load_float(a.teacher, l.base + k * l.stride, a.teacher_dtype) - norm;
        const double pk = norm == -INFINITY ? 0.0 : exp(lp);
        P += pk;
        listed |= 1ull << i;
        float zk = 0.f;
#pragma unroll
        for (int c = 0; c < CM; ++c) {
            if (c == (int)i) { zk = x.z[c]; target[c] += (float)pk; }
        }
        if (LOSS && !(pk == 0.0)) sum += pk * (lp - (empty ? -INFINITY : ((double)zk - m_all) * a.inv_t - log_all));
    }
    double mass = a.tail ? P : (norm == -INFINITY ? 0.0 : 1.0), rest = 0.0, q_rest = 1.0;
    float m_rest = m_all, s_rest = on.s;
    if (a.tail) {
        m_rest = -INFINITY;
#pragma unroll
        for (int c = 0; c < CM; ++c)
            if (!((listed >> c) & 1)) m_rest = fmaxf(m_rest, x.z[c]);
        const float refm = m_rest == -INFINITY ? 0.f : m_rest;
        s_rest = 0.f;
        float s_list = 0.f;
        const float ref_all = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
        for (int c = 0; c < CM; ++c) {
            const bool in = (listed >> c) & 1;
            const float e = exp2_hw((x.z[c] - (in ? ref_all : refm)) * a.c);
            s_rest += in ? 0.f : e;
            s_list += in ? e : 0.f;
        }
        if (s_rest > 0.f) {
            rest = P < 1.0 ? 1.0 - P : 0.0;
            mass = P + rest;
            double lq = 0.0;
            if (s_list > 0.f) {
                const double u = ((double)m_all - m_rest) * a.inv_t + log((double)s_list / s_rest);
                lq = -(u > 700.0 ? u : log1p(exp(u)));
            }
            q_rest = exp(lq);
            if (LOSS && rest > 0.0) sum += rest * (log(rest) - lq);
        }
    }
    if (bad) sum = NAN;
    if (LOSS) a.loss[r] = w == 0.f ? 0.f : (float)((on.s != on.s ? NAN : sum * a.t * a.t)) * w;
    if (GRAD) {
        const float up = (a.g_loss ? a.g_loss[r] : 1.f) * w;
        const float scale = up * a.t;
        const bool none = empty || (a.weight && w == 0.f);
        const float inv_all = 1.0f / on.s, inv_rest = s_rest > 0.f ? (float)((mass * q_rest - rest) / s_rest) : 0.f;
        const float ref_all = m_all == -INFINITY ? 0.f : m_all, ref_rest = m_rest == -INFINITY ? 0.f : m_rest;
        const float fm = (float)mass;
        T* out = grad + grad_start(v, p, r);
        const int64_t step = v.class_last ? 1 : v.inner;
#pragma unroll
        for (int c = 0; c < CM; ++c) {
            if (c < classes) {
                const bool in = !a.tail || ((listed >> c) & 1);
                const float e = exp2_hw((x.z[c] - (in ? ref_all : ref_rest)) * a.c);
                const float d = in ? fmaf(fm * inv_all, e, -target[c]) : inv_rest * e;
                out[c * step] = from_f32<T>(none ? 0.f : (bad || on.s != on.s ? NAN : scale * d));
            }
        }
    }
}

}  // namespace

// ---- launchers ---------------------------------------------------------------------------------------------------------------------------
namespace {
int vec_elems(int dtype) { return dtype == MICA_F32 ? 4 : 8; }
}  // namespace

bool score_is_col(const LogitsView& v) { return v.classes <= SCORE_COL_MAX; }

// Rows of up to WAVE_MAX classes take a wave each, longer ones a block.
static bool wave_rows(const LogitsView& v) { return v.classes <= 4096; }

// Few long rows: cut so that about 512 blocks have work, no segment below 8192 classes
SegPlan score_segments(const LogitsView& v, int64_t rows) {
    SegPlan s;
    s.n = 1;
    s.len = (int)v.classes;
    if (wave_rows(v)) return s;
    int64_t n = rows >= 512 ? 1 : 512 / rows;
    n = std::min<int64_t>(n, (v.classes + 4095) / 4096);
    n = std::max<int64_t>(n, (v.classes + SCORE_SEG_MAX - 1) / SCORE_SEG_MAX);
    if (n <= 1) return s;
    int64_t len = (v.classes + n - 1) / n;
    len = (len + 511) / 512 * 512;                          // 16-byte vectors of a segment begin where the row's do; bitmap words too
    s.len = (int)len;
    s.n = (int)((v.classes + len - 1) / len);
    return s;
}

template <typename F> static void by_dtype(int dtype, F&& f) {
    if (dtype == MICA_F32) f((float*)nullptr);
    else if (dtype == MICA_BF16) f((bf16_t*)nullptr);
    else f((f16_t*)nullptr);
}
template <typename F> static void by_classes(int64_t c, F&& f) {
    if (c <= 8) f(std::integral_constant<int, 8>());
    else if (c <= 24) f(std::integral_constant<int, 24>());
    else if (c <= 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 64>());
}
static unsigned blocks_of(int64_t items, int per) { return (unsigned)((items + per - 1) / per); }

int64_t score_ws_bytes(const LogitsView& v, int64_t rows, int top) {
    if (score_is_col(v)) return 0;
    const SegPlan s = score_segments(v, rows);
    return s.n == 1 ? 0 : rows * s.n * ((int64_t)sizeof(Partial) + (top ? 64 * 8 : 0));
}

void launch_score(const LogitsView& v, int64_t rows, const void* tokens, int token_bytes, int64_t ignore, float temperature, int top,
                  float* logprob, float* entropy, float* lse, float* top_logprob, int* top_index, void* ws, hipStream_t st) {
    ScoreOut o{tokens, token_bytes, ignore, logprob, entropy, lse, top_logprob, top_index, top, LOG2E / temperature, 1.0f / temperature};
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        if (score_is_col(v)) {
            by_classes(v.classes, [&](auto cm) {
                hipLaunchKernelGGL((score_col_kernel<T, decltype(cm)::value>), dim3(blocks_of(rows, 256)), dim3(256), 0, st, v, rows, o);
            });
            return;
        }
        const SegPlan s = score_segments(v, rows);
        Partial* part = static_cast<Partial*>(ws);
        u64* part_top = reinterpret_cast<u64*>(part + rows * s.n);
        const int64_t items = rows * s.n;
        if (wave_rows(v)) {
            if (top) hipLaunchKernelGGL((score_row_kernel<T, 64, true>), dim3(blocks_of(items, 4)), dim3(256), 0, st, v, rows, o, s.n, s.len, part, part_top);
            else hipLaunchKernelGGL((score_row_kernel<T, 64, false>), dim3(blocks_of(items, 4)), dim3(256), 0, st, v, rows, o, s.n, s.len, part, part_top);
        } else {
            if (top) hipLaunchKernelGGL((score_row_kernel<T, 256, true>), dim3((unsigned)items), dim3(256), 0, st, v, rows, o, s.n, s.len, part, part_top);
            else hipLaunchKernelGGL((score_row_kernel<T, 256, false>), dim3((unsigned)items), dim3(256), 0, st, v, rows, o, s.n, s.len, part, part_top);
        }
        if (s.n > 1) {
            if (top) hipLaunchKernelGGL((score_join_kernel<T, true>), dim3((unsigned)rows), dim3(256), 0, st, v, o, s.n, part, part_top);
            else hipLaunchKernelGGL((score_join_kernel<T, false>), dim3((unsigned)rows), dim3(256), 0, st, v, o, s.n, part, part_top);
        }
    });
}

void launch_score_grad(const LogitsView& v, int64_t rows, const void* tokens, int token_bytes, int64_t ignore, float temperature, const float* lse,
                       const float* entropy, const float* g_logprob, const float* g_entropy, const float* g_lse, void* grad, hipStream_t st) {
    ScoreGrad o{tokens, token_bytes, ignore, lse, entropy, g_logprob, g_entropy, g_lse, LOG2E / temperature, 1.0f / temperature};
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
        if (g == 64) hipLaunchKernelGGL((score_grad_row_kernel<T, 64>), dim3(blocks_of(rows * chunks, 4)), dim3(256), 0, st, v, rows, o, chunks, out);
        else hipLaunchKernelGGL((score_grad_row_kernel<T, 256>), dim3((unsigned)(rows * chunks)), dim3(256), 0, st, v, rows, o, chunks, out);
    });
}

int64_t distill_ws_bytes(const LogitsView& v, int64_t rows, bool step) {
    if (score_is_col(v)) return 0;
    const SegPlan s = score_segments(v, rows);
    if (s.n == 1) return 0;
    return rows * s.n * (int64_t)sizeof(Partial) + (step ? rows * 16 : 0);
}

static void distill_loss_rows(const LogitsView& v, int64_t rows, const DistillArgs& a, void* ws, hipStream_t st) {
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        const SegPlan s = score_segments(v, rows);
        Partial* part = static_cast<Partial*>(ws);
        const int64_t items = rows * s.n;
        const unsigned per = 4u * (a.k + (a.tail ? (s.len + 31) / 32 : 0));
        if (wave_rows(v)) {
            if (a.tail) hipLaunchKernelGGL((distill_row_kernel<T, 64, true>), dim3(blocks_of(items, 4)), dim3(256), per * 4, st, v, rows, a, s.n, s.len, part);
            else hipLaunchKernelGGL((distill_row_kernel<T, 64, false>), dim3(blocks_of(items, 4)), dim3(256), per * 4, st, v, rows, a, s.n, s.len, part);
        } else {
            if (a.tail) hipLaunchKernelGGL((distill_row_kernel<T, 256, true>), dim3((unsigned)items), dim3(256), per, st, v, rows, a, s.n, s.len, part);
            else hipLaunchKernelGGL((distill_row_kernel<T, 256, false>), dim3((unsigned)items), dim3(256), per, st, v, rows, a, s.n, s.len, part);
        }
        if (s.n > 1) hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)rows), dim3(256), 4u * a.k, st, v, rows, a, s.n, part);
    });
}
static void distill_grad_rows(const LogitsView& v, int64_t rows, const DistillArgs& a, void* grad, hipStream_t st) {
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        T* out = static_cast<T*>(grad);
        const int g = wave_rows(v) ? 64 : 256, chunk = g * UNROLL * vec_elems(v.dtype);
        const int chunks = (int)((v.classes + chunk - 1) / chunk);
        if (g == 64) hipLaunchKernelGGL((distill_grad_row_kernel<T, 64>), dim3(blocks_of(rows * chunks, 4)), dim3(256), 16u * a.k, st, v, rows, a, chunks, out);
        else hipLaunchKernelGGL((distill_grad_row_kernel<T, 256>), dim3((unsigned)(rows * chunks)), dim3(256), 4u * a.k, st, v, rows, a, chunks, out);
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
    a.inv_t = 1.0f / temperature;
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
    const SegPlan s = score_segments(v, rows);
    if (s.n > 1) {                                          // few long rows: the segments' sums first
        a.aux = reinterpret_cast<float*>(static_cast<Partial*>(ws) + rows * s.n);
        distill_loss_rows(v, rows, a, ws, st);
        distill_grad_rows(v, rows, a, grad, st);
        return;
    }
    by_dtype(v.dtype, [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        T* out = static_cast<T*>(grad);
        const unsigned per = 4u * (a.k + (a.tail ? (unsigned)((v.classes + 31) / 32) : 0));
        if (wave_rows(v)) {
            if (a.tail) hipLaunchKernelGGL((distill_step_row_kernel<T, 64, true>), dim3(blocks_of(rows, 4)), dim3(256), per * 4, st, v, rows, a, out);
            else hipLaunchKernelGGL((distill_step_row_kernel<T, 64, false>), dim3(blocks_of(rows, 4)), dim3(256), per * 4, st, v, rows, a, out);
        } else {
            if (a.tail) hipLaunchKernelGGL((distill_step_row_kernel<T, 256, true>), dim3((unsigned)rows), dim3(256), per, st, v, rows, a, out);
            else hipLaunchKernelGGL((distill_step_row_kernel<T, 256, false>), dim3((unsigned)rows), dim3(256), per, st, v, rows, a, out);
        }
    });
}

}  // namespace mica
