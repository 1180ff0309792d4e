// beam.hip -- beam selection over beams x buckets, and the beams' states
// reordered by parent.  The reference's look-ahead feeds one value seven times
// (ML/HTM/ModelTesting.py:66-72); a forecast that follows its own predictions
// keeps several continuations of every stream and drops the worse ones.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "beam_dev.h"
#include "htm_dev.h"

#define BS_MAX 64              // beams
#define BS_GROUPS (1 << 20)    // groups of one launch (of at most 1,024 threads each)

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(__hip_bfloat16 v) { return __bfloat162float(v); }

// ------------------------------------------------------------------ selection
// (score, place) as one unsigned key: larger is better, equal scores by the
// lower place; 0: never taken.  The upper word alone orders the scores.
__device__ __forceinline__ uint32_t score_bits(float s) {
    s += 0.0f;  // -0 and 0 are the same score
    if (!(s > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(s);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float bits_score(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

__device__ __forceinline__ uint64_t make_key(uint32_t bits, uint32_t place) {
    return bits ? ((uint64_t)bits << 32) | (0xFFFFFFFFu - place) : 0;
}

// a * b + c, c a constant in scalar registers.  (Left to itself the compiler moves
// every constant into the result's registers first, two instructions more.)
__device__ __forceinline__ double fma_s(double a, double b, double c) {
    asm("" : "+s"(c));
    return fma(a, b, c);
}

// exp(x - m) for finite m >= x, x = -infinity included (0), to a few units of 2^-53 as
// any float64 exponential: 2^t as 2^n 2^f, |f| <= 1/2, and 2^f as 1 + f q(f), q the
// polynomial of degree 10 through (2^f - 1) / f at the 11 Chebyshev nodes (off by 0.2 *
// 2^-53 with these coefficients).
__device__ __forceinline__ double exp_diff(float x, double m) {
    const double t = fmax(((double)x - m) * 1.4426950408889634074, -1100.0);
    const double n = rint(t), f = t - n;
    double p = 4.4549605981865186e-10;
    p = fma_s(p, f, 7.072585949269223e-09);
    p = fma_s(p, f, 1.0178062445845774e-07);
    p = fma_s(p, f, 1.321544258792169e-06);
    p = fma_s(p, f, 1.525273382983612e-05);
    p = fma_s(p, f, 1.540353044173605e-04);
    p = fma_s(p, f, 1.3333558146416936e-03);
    p = fma_s(p, f, 9.618129107606888e-03);
    p = fma_s(p, f, 5.55041086648216e-02);
    p = fma_s(p, f, 0.24022650695910097);
    p = fma_s(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}

__device__ __forceinline__ float wave_max(float v) {
    // lanes that a move does not reach take -infinity
    const auto step = [&](auto ctrl, auto rows) {
        const float o = __int_as_float(__builtin_amdgcn_update_dpp((int)0xFF800000, __float_as_int(v), decltype(ctrl)::value,
                                                                   decltype(rows)::value, 0xF, false));
        v = fmaxf(v, o);
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>(), integral_constant<int, 0xF>());  // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());  // row_bcast 15, 31
    step(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ double wave_sum(double v) {
    // lanes that a move does not reach take 0
    const auto step = [&](auto ctrl, auto rows) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, decltype(ctrl)::value,
                                                                  decltype(rows)::value, 0xF, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), decltype(ctrl)::value,
                                                                  decltype(rows)::value, 0xF, false);
        v += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>(), integral_constant<int, 0xF>());  // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());  // row_bcast 15, 31
    step(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// log(s) for s > 0: float32's, and the first terms of log(1 + d), d = s exp(-that) - 1
// some 1e-7.
__device__ __forceinline__ double log_of(double s) {
    const double y = (double)logf((float)s), d = s * exp_diff((float)-y, 0.0) - 1.0;
    return y + d * (1.0 - 0.5 * d);
}

__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A selection's LDS: the waves' best of each class, the list and its length.
struct TopSh {
    uint64_t* tops;  // [waves * 64]
    uint64_t* list;  // [room]
    uint32_t* count;
    int room;
};

// The best `want` (<= 64) of a workgroup's candidates.  mine: the thread's best
// key (0: none); each(f): f(key) for every candidate of the thread.  The lanes
// fall into 2^k >= want classes: the smallest of the classes' best is a floor that
// at least `want` candidates reach, and seldom many more (want H(want) if they lie
// anyhow), which are listed and count those before them.  Where more reach it
// than the list holds, or a class is empty, the best key below the last one is
// sought want times instead.  put(rank, key) is called once for each candidate
// taken; returns how many there are.  Every step compares distinct keys: the
// result does not depend on the order in which the list was filled.
template <typename EACH, typename PUT>
__device__ __forceinline__ int top_of(uint64_t mine, int want, const TopSh& sh, EACH each, PUT put) {
    const int nt = blockDim.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nwave = nt >> 6;
    int classes = 1;
    while (classes < want) classes *= 2;
    uint64_t best = mine;
    for (int k = 32; k >= classes; k >>= 1) best = max_key(best, __shfl_xor((unsigned long long)best, k));
    if (lane < classes) sh.tops[wave * classes + lane] = best;
    if (threadIdx.x == 0) *sh.count = 0;
    __syncthreads();
    uint64_t floor = 0;
    for (int w = 0; w < nwave; w++) floor = max_key(floor, sh.tops[w * classes + (lane & (classes - 1))]);
    {
        const uint32_t hi = ~wave_max_u32(~(uint32_t)(floor >> 32));
        const uint32_t lo = ~wave_max_u32((uint32_t)(floor >> 32) == hi ? ~(uint32_t)floor : 0u);
        floor = hi ? ((uint64_t)hi << 32) | lo : 1;
    }
    if (mine >= floor)
        each([&](uint64_t k) {
            if (k >= floor) {
                const uint32_t at = atomicAdd(sh.count, 1u);
                if (at < (uint32_t)sh.room) sh.list[at] = k;
            }
        });
    __syncthreads();
    const int m = (int)*sh.count;
    if (m <= sh.room) {
        for (int i = threadIdx.x; i < m; i += nt) {
            const uint64_t k = sh.list[i];
            int before = 0;
#pragma unroll 4
            for (int j = 0; j < m; j++) before += sh.list[j] > k ? 1 : 0;
            if (before < want) put(before, k);
        }
        return min(m, want);
    }
    uint64_t prev = ~0ull;
    for (int r = 0; r < want; r++) {
        best = 0;
        each([&](uint64_t k) {
            if (k < prev && k > best) best = k;
        });
        // the upper word's largest, then the lower word's among those
        const uint32_t hi = wave_max_u32((uint32_t)(best >> 32));
        const uint32_t lo = wave_max_u32((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        if (lane == 0) sh.tops[wave] = ((uint64_t)hi << 32) | lo;
        __syncthreads();
        best = 0;
        for (int w = 0; w < nwave; w++) best = max_key(best, sh.tops[w]);
        __syncthreads();
        if (!best) return r;
        if (threadIdx.x == 0) put(r, best);
        prev = best;
    }
    return want;
}

struct SelArgs {
    const void* x;
    int64_t gs, bs;
    const float* score;
    const int32_t* live;
    int64_t g0;  // the launch's first group
    int32_t win, wout, v;
    float* o_score;
    int32_t* o_parent;
    int32_t* o_bucket;
};

__device__ __forceinline__ int live_of(const SelArgs& a, int64_t g) {
    return a.live ? min(max(a.live[g], 0), a.v) : a.v;
}

__device__ __forceinline__ void put_key(const SelArgs& a, int64_t g, int rank, uint64_t k) {
    const int64_t at = g * a.wout + rank;
    const uint32_t place = 0xFFFFFFFFu - (uint32_t)k;
    a.o_score[at] = bits_score((uint32_t)(k >> 32));
    a.o_parent[at] = (int32_t)(place / (uint32_t)a.v);
    a.o_bucket[at] = (int32_t)(place % (uint32_t)a.v);
}

__device__ __forceinline__ void put_rest(const SelArgs& a, int64_t g, int taken) {
    for (int r = taken + (int)threadIdx.x; r < a.wout; r += blockDim.x) {
        const int64_t at = g * a.wout + r;
        a.o_score[at] = -INFINITY;
        a.o_parent[at] = min(r, a.win - 1);
        a.o_bucket[at] = -1;
    }
}

// Up to 1,024 outputs a beam: one workgroup per group, a wave for each R beams,
// whose up to E * 64 outputs stay in registers from the load to the selection,
// and no barrier before it.  What it costs is the chain of one wave: load, the
// largest, E exponentials, the sum, a logarithm, the scores.  Measured, us, 8 x
// 480 -> 8: one group 5.6 (the logits in LDS, between barriers: 10.4), 512 groups
// 8.2 (13.6), 4,096 groups 30 to 34 (54); two beams a wave 7.0, 9.0, 33.  Many groups
// are bound by instructions, most of them float64: 1.7e7 of a wave, 510 for each
// beam, are 31 us of issue at the 4.5 cycles that one takes; the 63 MB take 13.
template <typename T, int R, int E>
__global__ void __launch_bounds__(1024) beam_small_kernel(SelArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint64_t small_sh[];  // tops, list: 64 a wave each
    __shared__ uint32_t count;
    const TopSh sh{small_sh, small_sh + blockDim.x, &count, (int)blockDim.x};
    const int64_t g = a.g0 + blockIdx.x;
    const int lane = threadIdx.x & 63, w0 = (threadIdx.x >> 6) * R;
    const int n = live_of(a, g);
    const T* x = (const T*)a.x + g * a.gs;
    T in[R][E];  // (every read without a branch and a conversion, which would wait for it)
    float v[R][E], m[R];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int e = 0; e < E; e++) in[r][e] = x[min(w0 + r, a.win - 1) * a.bs + min(e * 64 + lane, a.v - 1)];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int e = 0; e < E; e++) v[r][e] = w0 + r < a.win && e * 64 + lane < n ? up(in[r][e]) : -INFINITY;
    float best = -INFINITY;
    uint32_t at = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        m[r] = -INFINITY;
        bool nan = false;
#pragma unroll
        for (int e = 0; e < E; e++) {
            m[r] = fmaxf(m[r], v[r][e]);
            nan |= v[r][e] != v[r][e];
        }
        m[r] = wave_max(nan ? INFINITY : m[r]);  // (a NaN spoils the beam as +infinity does)
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool fine = fabsf(m[r]) < INFINITY;
        const double md = fine ? (double)m[r] : 0.0;
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (e * 64 < n) s += exp_diff(v[r][e], md);  // (the same branch for the whole wave)
        s = wave_sum(s);
        // (no finite logit, an infinite one or a NaN: no score of the beam is a number)
        const double base = fine ? (double)a.score[g * a.win + w0 + r] - log_of(s) : (double)NAN;
#pragma unroll
        for (int e = 0; e < E; e++) {
            v[r][e] = (float)(((double)v[r][e] - md) + base);
            if (v[r][e] > best) best = v[r][e], at = (uint32_t)(w0 + r) << 16 | (uint32_t)(e * 64 + lane);
        }
    }
    // (a place in the key: beam and output in 16 bits each, in the same order)
    const auto each = [&](auto f) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int e = 0; e < E; e++) f(make_key(score_bits(v[r][e]), (uint32_t)(w0 + r) << 16 | (uint32_t)(e * 64 + lane)));
    };
    const int taken = top_of(make_key(score_bits(best), at), a.wout, sh, each, [&](int r, uint64_t k) {
        const uint32_t place = 0xFFFFFFFFu - (uint32_t)k;
        const int64_t o = g * a.wout + r;
        a.o_score[o] = bits_score((uint32_t)(k >> 32));
        a.o_parent[o] = (int32_t)(place >> 16);
        a.o_bucket[o] = (int32_t)(place & 0xFFFFu);
    });
    put_rest(a, g, taken);
}

// More (beams_in * n_outputs <= BS_ONE): one workgroup per group, the logits read
// once into LDS.  parts waves share a beam.  100 groups of 4 x 2,000: 12.7 us, the chain of
// the same steps with a barrier behind each.
#define BS_ONE 8192
#define BS_LIST 512
template <typename T>
__global__ void __launch_bounds__(1024) beam_select_kernel(SelArgs a, int parts, uint32_t inv_v) {
    __shared__ uint32_t count;
    __shared__ double sum[BS_MAX];   // [beam * parts + part]: parts > 1 only while beams * parts <= waves
    __shared__ float top[BS_MAX];
    __shared__ double base[BS_MAX];  // a beam's score - log(sum); NaN: none of its continuations counts
    __shared__ double largest[BS_MAX];  // its largest logit
    extern __shared__ __attribute__((aligned(16))) uint64_t select_sh[];  // tops, list, [win * v] logits, then scores
    const TopSh sh{select_sh, select_sh + blockDim.x, &count, BS_LIST};
    float* cand = reinterpret_cast<float*>(select_sh + blockDim.x + BS_LIST);
    const int64_t g = a.g0 + blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nwave = blockDim.x >> 6;
    const int n = live_of(a, g), rows = nwave / parts, part = wave % parts, first = wave / parts;
    const T* x = (const T*)a.x + g * a.gs;
    const int step = parts * 64, o0 = part * 64 + lane;
    const int all = a.win * a.v;
    for (int i0 = threadIdx.x; i0 < all; i0 += 16 * blockDim.x) {  // 16 loads of a thread under way at once
        T v[16];
        bool live[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int i = min(i0 + j * (int)blockDim.x, all - 1);
            const int w = a.v == 1 ? i : (int)__umulhi((uint32_t)i, inv_v), o = i - w * a.v;
            v[j] = x[(int64_t)w * a.bs + o];  // (without a branch and a conversion, which would wait for it)
            live[j] = o < n;
        }
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (i0 + j * (int)blockDim.x < all) cand[i0 + j * blockDim.x] = live[j] ? up(v[j]) : -INFINITY;
    }
    __syncthreads();
    // eight of a beam's outputs a lane at a time, -infinity behind the live ones
    const auto eight = [&](const float* c, int o, float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = o + j * step < n ? c[o + j * step] : -INFINITY;
    };
    for (int w = first; w < a.win; w += rows) {
        float m = -INFINITY;
        bool nan = false;
        for (int o = o0; o - lane < n; o += 8 * step) {
            float v[8];
            eight(cand + w * a.v, o, v);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                m = fmaxf(m, v[j]);
                nan |= v[j] != v[j];
            }
        }
        m = wave_max(nan ? INFINITY : m);  // (a NaN spoils the beam as +infinity does)
        if (lane == 0) top[w * parts + part] = m;
    }
    __syncthreads();
    for (int w = first; w < a.win; w += rows) {
        float m = top[w * parts];
        for (int k = 1; k < parts; k++) m = fmaxf(m, top[w * parts + k]);
        const double md = (double)m;
        double s[2] = {0.0, 0.0};
        if (fabsf(m) < INFINITY)
            for (int o = o0; o - lane < n; o += 8 * step) {
                float v[8];
                eight(cand + w * a.v, o, v);
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    if (o - lane + j * step < n) {  // (the same for the whole wave)
                        s[0] += exp_diff(v[j], md);
                        s[1] += exp_diff(v[j + 1], md);
                    }
            }
        s[0] = wave_sum(s[0] + s[1]);
        if (lane == 0) sum[w * parts + part] = s[0];
    }
    __syncthreads();
    if ((int)threadIdx.x < a.win) {
        const int w = threadIdx.x;
        float m = top[w * parts];
        double s = sum[w * parts];
        for (int k = 1; k < parts; k++) {
            m = fmaxf(m, top[w * parts + k]);
            s += sum[w * parts + k];
        }
        largest[w] = (double)m;
        // (no finite logit, an infinite one or a NaN: no score of the beam is a number)
        base[w] = fabsf(m) < INFINITY ? (double)a.score[g * a.win + w] - log_of(s) : (double)NAN;
    }
    __syncthreads();
    float best = -INFINITY;
    uint32_t at = 0;
    for (int w = first; w < a.win; w += rows) {
        const double b = base[w], m = largest[w];
        float* c = cand + w * a.v;
        for (int o = o0; o - lane < n; o += 8 * step) {
            float v[8];
            eight(c, o, v);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (o + j * step < n) {
                    v[j] = (float)(((double)v[j] - m) + b);
                    c[o + j * step] = v[j];
                    if (v[j] > best) best = v[j], at = (uint32_t)(w * a.v + o + j * step);
                }
        }
    }
    const auto each = [&](auto f) {
        for (int w = first; w < a.win; w += rows)
            for (int o = o0; o - lane < n; o += 8 * step) {
                float v[8];
                eight(cand + w * a.v, o, v);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (v[j] > -INFINITY) f(make_key(score_bits(v[j]), (uint32_t)(w * a.v + o + j * step)));
            }
    };
    const int taken = top_of(make_key(score_bits(best), at), a.wout, sh, each, [&](int r, uint64_t k) { put_key(a, g, r, k); });
    put_rest(a, g, taken);
}

// Many candidates: chunks of BS_CHUNK of a beam's outputs, three launches, since a
// beam's sum is needed before its first score.  4 groups of 16 x 32,768 bfloat16 -> 16:
// 5.8, 11 and 6 us in 21 us, each the latency of a few loads, sums and a selection;
// the 4 MB of logits are read again from the caches.
#define BS_CHUNK 4096
struct SelWork {
    float* top;      // [groups * win * chunks] the chunks' largest logits, +infinity where there is a NaN
    double* sum;     // ... and sums of exp(x - top)
    uint64_t* keys;  // [groups * win * chunks * wout] the chunks' best
    int32_t chunks;
};

// A thread's logits of a chunk, -infinity behind the live ones.  Every read without a
// branch and a conversion, which would wait for it.
template <typename T>
__device__ __forceinline__ void chunk_logits(const T* p, int o0, int n, int all, float (&v)[BS_CHUNK / 256]) {
    T in[BS_CHUNK / 256];
#pragma unroll
    for (int j = 0; j < BS_CHUNK / 256; j++) in[j] = p[min(o0 + j * 256 + (int)threadIdx.x, all - 1)];
#pragma unroll
    for (int j = 0; j < BS_CHUNK / 256; j++) v[j] = o0 + j * 256 + (int)threadIdx.x < n ? up(in[j]) : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(256) beam_sums_kernel(SelArgs a, SelWork k, int64_t row0) {
    __shared__ float tm[4];
    __shared__ double ts[4];
    const int64_t row = row0 + blockIdx.y, g = row / a.win;
    const int o0 = blockIdx.x * BS_CHUNK, n = min(live_of(a, g), o0 + BS_CHUNK);
    const T* p = (const T*)a.x + g * a.gs + (row - g * a.win) * a.bs;
    float v[BS_CHUNK / 256], m = -INFINITY;
    bool nan = false;
    chunk_logits(p, o0, n, a.v, v);
#pragma unroll
    for (int j = 0; j < BS_CHUNK / 256; j++) {
        m = fmaxf(m, v[j]);
        nan |= v[j] != v[j];
    }
    m = wave_max(nan ? INFINITY : m);
    if ((threadIdx.x & 63) == 0) tm[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]));
    const double md = (double)m;
    double s = 0.0;
    if (fabsf(m) < INFINITY) {
#pragma unroll 4
        for (int j = 0; j < BS_CHUNK / 256; j++) s += exp_diff(v[j], md);
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) ts[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        k.top[row * k.chunks + blockIdx.x] = m;
        k.sum[row * k.chunks + blockIdx.x] = (ts[0] + ts[1]) + (ts[2] + ts[3]);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) beam_chunk_kernel(SelArgs a, SelWork k, int64_t row0) {
    __shared__ uint64_t tops[4 * 64], list[1024];
    __shared__ uint32_t count;
    const TopSh sh{tops, list, &count, 1024};
    __shared__ float tm[4];
    __shared__ double ts[4];
    const int64_t row = row0 + blockIdx.y, g = row / a.win;
    const int o0 = blockIdx.x * BS_CHUNK, n = min(live_of(a, g), o0 + BS_CHUNK), w = (int)(row - g * a.win);
    const T* p = (const T*)a.x + g * a.gs + w * a.bs;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float v[BS_CHUNK / 256];
    chunk_logits(p, o0, n, a.v, v);
    // the beam's largest logit and sum from its chunks'
    const float* top = k.top + row * k.chunks;
    const double* sum = k.sum + row * k.chunks;
    float m = -INFINITY;
    for (int c = threadIdx.x; c < k.chunks; c += 256) m = fmaxf(m, top[c]);
    m = wave_max(m);
    if (lane == 0) tm[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]));
    const double md = (double)m;
    double s = 0.0;
    if (fabsf(m) < INFINITY)
        for (int c = threadIdx.x; c < k.chunks; c += 256) s += sum[c] * exp_diff(top[c], md);
    s = wave_sum(s);
    if (lane == 0) ts[wave] = s;
    __syncthreads();
    s = (ts[0] + ts[1]) + (ts[2] + ts[3]);
    const double base = fabsf(m) < INFINITY ? (double)a.score[row] - log_of(s) : (double)NAN;
    float best = -INFINITY;
    uint32_t at = 0;
    const uint32_t place0 = (uint32_t)(w * (int64_t)a.v + o0);
#pragma unroll
    for (int j = 0; j < BS_CHUNK / 256; j++) {
        v[j] = (float)(((double)v[j] - md) + base);  // (behind the live outputs: -infinity or NaN)
        if (v[j] > best) best = v[j], at = place0 + j * 256 + threadIdx.x;
    }
    uint64_t* keys = k.keys + (row * k.chunks + blockIdx.x) * a.wout;
    const auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < BS_CHUNK / 256; j++) f(make_key(score_bits(v[j]), place0 + j * 256 + threadIdx.x));
    };
    // every chunk's ranks begin at another place: the merge's classes then hold all ranks and all beams, and their best
    // make a floor that few keys reach (in order, with beams alike, nearly all do: 4 groups of 16 x 32,768 -> 16 71 us
    // instead of 6)
    const int turn = (int)((w * (int64_t)k.chunks + blockIdx.x) % a.wout);
    const auto place = [&](int r) { return r + turn < a.wout ? r + turn : r + turn - a.wout; };
    const int taken = top_of(make_key(score_bits(best), at), a.wout, sh, each, [&](int r, uint64_t key) { keys[place(r)] = key; });
    for (int r = taken + (int)threadIdx.x; r < a.wout; r += 256) keys[place(r)] = 0;
}

// The chunks' best of one group: the best of them.
__global__ void __launch_bounds__(1024) beam_merge_kernel(SelArgs a, SelWork k) {
    __shared__ uint64_t tops[16 * 64], list[1024];
    __shared__ uint32_t count;
    const TopSh sh{tops, list, &count, 1024};
    const int64_t g = a.g0 + blockIdx.x;
    const uint32_t rows = (uint32_t)a.win * (uint32_t)k.chunks, n = rows * (uint32_t)a.wout;  // (at most 2^24 + 4,096)
    const uint64_t* keys = k.keys + g * n;
    uint64_t best = 0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) best = max_key(best, keys[i]);
    const auto each = [&](auto f) {
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) f(keys[i]);
    };
    put_rest(a, g, top_of(best, a.wout, sh, each, [&](int r, uint64_t k) { put_key(a, g, r, k); }));
}

// ------------------------------------------------------------------- rows
// All buffers of a call in one launch: block b belongs to buffer k with first[k]
// <= b < first[k + 1].  A buffer's rows are moved in its widest unit (16 bytes
// down to 1, what its size and addresses divide by); 2^lanes[k] threads share a
// row, four units each, all read before the first is written.  Bound by memory:
// 32,768 rows of 9,856 B, 8 beams a group, parents at random: 109 us for 535 MB read
// and written, 4.9 TB/s, as fast as a plain copy; 323 MB of a fleet's states, some 30 KB
// a row over several buffers, 62 us.
struct MoveArgs {
    RowMoves m;
    uint32_t first[HTM_BEAM_BUFFERS + 1];
    uint32_t units[HTM_BEAM_BUFFERS];   // of a row
    uint8_t width[HTM_BEAM_BUFFERS];    // log2 of a unit's bytes
    uint8_t lanes[HTM_BEAM_BUFFERS];
    uint16_t parts[HTM_BEAM_BUFFERS];   // blocks side by side over a row
    const int32_t* idx;
    int64_t n_rows, n_src;
    int32_t beams;
};

#define MOVE_UNITS 4
typedef uint32_t unit16 __attribute__((ext_vector_type(4)));
typedef uint32_t unit8 __attribute__((ext_vector_type(2)));

template <typename U>
__device__ __forceinline__ void move_out(const MoveArgs& a, int k, uint32_t block) {
    const int log = a.lanes[k], t = threadIdx.x & ((1 << log) - 1);
    const uint32_t units = a.units[k], parts = a.parts[k];
    const uint32_t row_block = parts == 1 ? block : block / parts, part = block - row_block * parts;
    const int64_t r = ((int64_t)row_block << (8 - log)) + (threadIdx.x >> log);
    if (r >= a.n_rows) return;
    int64_t from = a.idx[r];
    if (a.beams) {
        const int64_t w = a.n_rows <= 0xFFFFFFFFll ? (int64_t)((uint32_t)r % (uint32_t)a.beams) : r % a.beams;
        from = r - w + (from >= 0 && from < a.beams ? from : w);
    } else if (from < 0 || from >= a.n_src) {
        return;
    }
    const U* src = reinterpret_cast<const U*>(a.m.src[k]) + from * (int64_t)units;
    U* dst = reinterpret_cast<U*>(a.m.dst[k]) + r * (int64_t)units;
    const uint32_t u0 = part * (MOVE_UNITS * 256) + t;
    U v[MOVE_UNITS];
#pragma unroll
    for (int j = 0; j < MOVE_UNITS; j++)
        if (u0 + (j << log) < units) v[j] = src[u0 + (j << log)];
#pragma unroll
    for (int j = 0; j < MOVE_UNITS; j++)
        if (u0 + (j << log) < units) dst[u0 + (j << log)] = v[j];
}

__device__ __forceinline__ int move_buffer(const MoveArgs& a) {
    int k = 0;
    while (blockIdx.x >= a.first[k + 1]) k++;
    return k;
}

// Blocks go to the chip's 8 XCDs in turn; each takes a run of neighbouring rows,
// so that a parent of several rows of a group is read from memory once, into
// the L2 of the XCD that copies the group.
__device__ __forceinline__ uint32_t near_block(uint32_t b, uint32_t n) {
    const uint32_t q = n / 8, r = n % 8, x = b % 8, i = b / 8;
    return x * q + min(x, r) + i;
}

__global__ void __launch_bounds__(256) rows_copy_kernel(MoveArgs a) {
    const int k = move_buffer(a);
    const uint32_t b = near_block(blockIdx.x - a.first[k], a.first[k + 1] - a.first[k]);
    if (a.width[k] == 4) move_out<unit16>(a, k, b);
    else if (a.width[k] == 3) move_out<unit8>(a, k, b);
    else if (a.width[k] == 2) move_out<uint32_t>(a, k, b);
    else if (a.width[k] == 1) move_out<uint16_t>(a, k, b);
    else move_out<uint8_t>(a, k, b);
}

// In place: a thread owns a unit's place in all W rows of a group, reads the
// parents' and only then writes, so that no other thread's data is involved and
// nothing is kept beside the buffers.  Rows that stay are not touched.  The same rows
// as above, only those that move written: 2 beams 115 us, 8 92 us (5.4 TB/s), 16 103
// us, 32 126 us, 64 187 us (2.8 TB/s): the more rows a thread holds, the fewer waves
// a CU does.
template <typename U, int W>
__device__ __forceinline__ void move_in(const MoveArgs& a, int k, uint32_t block) {
    const int log = a.lanes[k], t = threadIdx.x & ((1 << log) - 1);
    const uint32_t units = a.units[k], parts = a.parts[k];
    const uint32_t row_block = parts == 1 ? block : block / parts, part = block - row_block * parts;
    const int64_t g = ((int64_t)row_block << (8 - log)) + (threadIdx.x >> log);
    const uint32_t u = part * 256 + t;
    if (g >= a.n_rows / a.beams || u >= units) return;
    const int32_t* p = a.idx + g * a.beams;
    U* b = reinterpret_cast<U*>(a.m.dst[k]) + g * a.beams * (int64_t)units + u;
    // (a row that stays reads row 0 instead: a read without a branch, of a row that is read at most once more)
    U v[W];
    uint64_t moved = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int q = w < a.beams ? p[w] : w;
        const bool go = q >= 0 && q < a.beams && q != w;
        moved |= (uint64_t)go << w;
        v[w] = b[(uint64_t)(go ? (uint32_t)q : 0u) * units];
    }
#pragma unroll
    for (int w = 0; w < W; w++)
        if ((moved >> w) & 1) b[(uint64_t)w * units] = v[w];
}

template <int W>
__global__ void __launch_bounds__(256, W <= 8 ? 8 : W <= 32 ? 5 : 2) rows_inplace_kernel(MoveArgs a) {
    const int k = move_buffer(a);
    const uint32_t b = blockIdx.x - a.first[k];
    if (W <= 16 && a.width[k] == 4) move_in<unit16, (W <= 16 ? W : 1)>(a, k, b);
    else if (a.width[k] == 3) move_in<unit8, W>(a, k, b);
    else if (a.width[k] == 2) move_in<uint32_t, W>(a, k, b);
    else if (a.width[k] == 1) move_in<uint16_t, W>(a, k, b);
    else move_in<uint8_t, W>(a, k, b);
}

int rows_move(const RowMoves& m, const int32_t* idx, int64_t n_rows, int32_t beams, int64_t n_src, hipStream_t st) {
    if (!n_rows) return HTM_OK;
    for (int inplace = 0; inplace < (beams ? 2 : 1); inplace++) {  // (an index of rows, beams 0, never moves in place)
        MoveArgs a;
        a.m.n = 0;
        a.idx = idx;
        a.n_rows = n_rows;
        a.n_src = n_src;
        a.beams = beams;
        uint64_t blocks = 0;
        const int64_t items = inplace ? n_rows / beams : n_rows;
        for (int k = 0; k < m.n; k++) {
            if (!m.bytes[k] || (m.src[k] == m.dst[k]) != (inplace != 0)) continue;
            const int i = a.m.n++;
            a.m.src[i] = m.src[k];
            a.m.dst[i] = m.dst[k];
            a.m.bytes[i] = m.bytes[k];
            const uint64_t all = m.bytes[k] | (uint64_t)(uintptr_t)m.src[k] | (uint64_t)(uintptr_t)m.dst[k];
            // (more than 16 beams in place: 8-byte units halve a thread's registers; 32 beams 126 us, by 16 bytes 139)
            int width = inplace && beams > 16 ? 3 : 4;
            while (width && all & ((1ull << width) - 1)) width--;
            const uint64_t units = m.bytes[k] >> width, per = inplace ? 1 : MOVE_UNITS;
            int lanes = 0;
            while (lanes < 8 && (per << lanes) < units) lanes++;
            const uint64_t parts = (units + (per << 8) - 1) / (per << 8);
            const uint64_t add = (((uint64_t)items + (256u >> lanes) - 1) >> (8 - lanes)) * parts;
            if (units > 0xFFFFFFFFull || parts > 0xFFFFull || blocks + add > 0xFFFFFFull)
                return htm_fail(HTM_E_INVALID, "rows of %llu bytes x %lld are more than one launch moves",
                                (unsigned long long)m.bytes[k], (long long)n_rows);
            a.units[i] = (uint32_t)units;
            a.width[i] = (uint8_t)width;
            a.lanes[i] = (uint8_t)lanes;
            a.parts[i] = (uint16_t)parts;
            a.first[i] = (uint32_t)blocks;
            blocks += add;
            a.first[i + 1] = (uint32_t)blocks;
        }
        if (!blocks) continue;
        const dim3 grid((uint32_t)blocks);
        if (!inplace) hipLaunchKernelGGL(rows_copy_kernel, grid, dim3(256), 0, st, a);
        else if (beams <= 8) hipLaunchKernelGGL(rows_inplace_kernel<8>, grid, dim3(256), 0, st, a);
        else if (beams <= 16) hipLaunchKernelGGL(rows_inplace_kernel<16>, grid, dim3(256), 0, st, a);
        else if (beams <= 32) hipLaunchKernelGGL(rows_inplace_kernel<32>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(rows_inplace_kernel<64>, grid, dim3(256), 0, st, a);
    }
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "row move launch failed");
}

extern "C" {

// a beam's outputs fit a wave's registers, and 16 waves the beams
static bool sel_small(int32_t win, int32_t v) { return v <= 1024 && win <= (v <= 256 ? 64 : v <= 512 ? 32 : 16); }

static int sel_chunks(int32_t v) { return (v + BS_CHUNK - 1) / BS_CHUNK; }

size_t htm_beam_work_bytes(int32_t groups, int32_t win, int32_t wout, int32_t v) {
    if (groups < 1 || win < 1 || win > BS_MAX || wout < 1 || wout > BS_MAX || v < 1 || sel_small(win, v) ||
        (int64_t)win * v <= BS_ONE)
        return 0;
    return (size_t)groups * win * sel_chunks(v) * (8 + 8 + 8 * (size_t)wout);
}

}  // extern "C"

template <typename T>
static void select_launch(SelArgs a, int32_t groups, void* work, hipStream_t st) {
    const int64_t all = (int64_t)a.win * a.v;
    const bool small = sel_small(a.win, a.v);
    SelWork k{};
    if (!small && all > BS_ONE) {
        k.chunks = sel_chunks(a.v);
        const int64_t rows = (int64_t)groups * a.win;
        k.sum = (double*)work;
        k.keys = (uint64_t*)(k.sum + rows * k.chunks);
        k.top = (float*)(k.keys + rows * k.chunks * a.wout);
        for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
            const dim3 grid(k.chunks, (uint32_t)(rows - r0 < 65535 ? rows - r0 : 65535));
            hipLaunchKernelGGL(beam_sums_kernel<T>, grid, dim3(256), 0, st, a, k, r0);
            hipLaunchKernelGGL(beam_chunk_kernel<T>, grid, dim3(256), 0, st, a, k, r0);
        }
    }
    for (int64_t g0 = 0; g0 < groups; g0 += BS_GROUPS) {
        a.g0 = g0;
        const dim3 grid((uint32_t)(groups - g0 < BS_GROUPS ? groups - g0 : BS_GROUPS));
        if (small) {
            const int each = (a.win + 15) / 16, waves = each > 2 ? (a.win + 3) / 4 : (a.win + each - 1) / each;
            const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(waves * 64), waves * 64 * 16, st, a); };
            if (each > 2) go(beam_small_kernel<T, 4, 4>);
            else if (each == 2) a.v <= 256 ? go(beam_small_kernel<T, 2, 4>) : go(beam_small_kernel<T, 2, 8>);
            else if (a.v <= 256) go(beam_small_kernel<T, 1, 4>);
            else if (a.v <= 512) go(beam_small_kernel<T, 1, 8>);
            else go(beam_small_kernel<T, 1, 16>);
        } else if (all <= BS_ONE) {
            // (100 groups of 4 x 2,000: 256 threads 15.2 us, 512 12.7, 1,024 13.3; 2,000 groups: 39, 42, 90)
            const int nt = groups < 512 ? 512 : 256;
            int parts = 1;
            while (parts * 2 * a.win <= nt / 64) parts *= 2;
            const size_t lds = (size_t)(nt + BS_LIST) * sizeof(uint64_t) + (size_t)all * sizeof(float);
            hipLaunchKernelGGL(beam_select_kernel<T>, grid, dim3(nt), lds, st, a, parts, 0xFFFFFFFFu / (uint32_t)a.v + 1u);
        } else {
            const int64_t keys = (int64_t)a.win * k.chunks * a.wout;
            hipLaunchKernelGGL(beam_merge_kernel, grid, dim3(keys > 2048 ? 1024 : 256), 0, st, a, k);
        }
    }
}

extern "C" {

int htm_beam_select(const void* x, int32_t dtype, int64_t gs, int64_t bs, const float* score, const int32_t* live,
                    int32_t groups, int32_t win, int32_t wout, int32_t v, float* o_score, int32_t* o_parent,
                    int32_t* o_bucket, void* work, size_t work_bytes, void* stream) {
    if (groups < 0 || win < 1 || win > BS_MAX || wout < 1 || wout > BS_MAX || v < 1 || (int64_t)win * v > (1ll << 30))
        return htm_fail(HTM_E_INVALID, "%s: 1..64 beams in and out, outputs >= 1, beams_in * outputs <= 2^30", __func__);
    if (dtype != HTM_T_F32 && dtype != HTM_T_F16 && dtype != HTM_T_BF16)
        return htm_fail(HTM_E_INVALID, "%s: d_logits must be float32, float16 or bfloat16", __func__);
    if (!groups) return HTM_OK;
    if (!x || !score || !o_score || !o_parent || !o_bucket || gs < 0 || bs < 0)
        return htm_fail(HTM_E_INVALID, "%s: invalid argument", __func__);
    const size_t need = htm_beam_work_bytes(groups, win, wout, v);
    if (need && (!work || (uintptr_t)work % 8 || work_bytes < need))
        return htm_fail(HTM_E_INVALID, "%s: needs htm_beam_work_bytes of scratch, 8-byte aligned", __func__);
    const SelArgs a{x, gs, bs, score, live, 0, win, wout, v, o_score, o_parent, o_bucket};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == HTM_T_F32) select_launch<float>(a, groups, work, st);
    else if (dtype == HTM_T_F16) select_launch<__half>(a, groups, work, st);
    else select_launch<__hip_bfloat16>(a, groups, work, st);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "beam select launch failed");
}

int htm_beam_reorder(int32_t n, const void* const* src, void* const* dst, const size_t* bytes, const int32_t* parent,
                     int32_t groups, int32_t beams, void* stream) {
    if (n < 1 || n > HTM_BEAM_BUFFERS || !src || !dst || !bytes || groups < 0 || beams < 1 || beams > BS_MAX)
        return htm_fail(HTM_E_INVALID, "%s: 1..%d buffers, 1..64 beams", __func__, HTM_BEAM_BUFFERS);
    const int64_t rows = (int64_t)groups * beams;
    if (!rows) return HTM_OK;
    if (!parent) return htm_fail(HTM_E_INVALID, "%s: null parents", __func__);
    RowMoves m;
    m.n = n;
    for (int k = 0; k < n; k++) {
        m.src[k] = (const uint8_t*)src[k];
        m.dst[k] = (uint8_t*)dst[k];
        m.bytes[k] = bytes[k];
        if (bytes[k] > ((size_t)1 << 40) / (size_t)rows) return htm_fail(HTM_E_INVALID, "%s: buffer %d too large", __func__, k);
        if (bytes[k] && (!src[k] || !dst[k])) return htm_fail(HTM_E_INVALID, "%s: null buffer %d", __func__, k);
    }
    // a destination may be its own source, and overlaps nothing else that is read or written here
    for (int k = 0; k < n; k++) {
        const uintptr_t d0 = (uintptr_t)dst[k], d1 = d0 + bytes[k] * (size_t)rows;
        for (int j = 0; j < n; j++) {
            const uintptr_t s0 = (uintptr_t)src[j], s1 = s0 + bytes[j] * (size_t)rows;
            const uintptr_t e0 = (uintptr_t)dst[j], e1 = e0 + bytes[j] * (size_t)rows;
            if ((d0 < s1 && s0 < d1 && !(j == k && s0 == d0)) || (j != k && d0 < e1 && e0 < d1))
                return htm_fail(HTM_E_INVALID, "%s: buffer %d overlaps buffer %d", __func__, k, j);
        }
        const uintptr_t p0 = (uintptr_t)parent, p1 = p0 + (size_t)rows * 4;
        if (d0 < p1 && p0 < d1) return htm_fail(HTM_E_INVALID, "%s: buffer %d overlaps the parents", __func__, k);
    }
    return rows_move(m, parent, rows, beams, rows, (hipStream_t)stream);
}

}  // extern "C"
