// readout.hip -- 4-bit matrix-vector products with group scales: a frozen
// SDRClassifier's answer (ML/HTM/NetworkModel.py:70-97 is the region whose
// float64 product this stands in for once learning is off), or any linear
// read-out of cells or columns.
//
//   y[r][h][o] = sum_i x[r][i] * scale[i][h][o / group] * (code[i][h][o] - 8)
//
// A record holds one input's weights of all heads, codes then scales, so that
// an active cell's contribution is one contiguous read.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "htm_dev.h"
#include "q4_dev.h"

#define Q4_NT 256
#define Q4_MAX_SCALE 1.2676506002282294e30  // 2^100: 65,536 weights' sum stays finite
#define Q4_MIN_SCALE 7.7037197775489434e-34 // 2^-110: its lower four bits are a normal number (q4_mfma_kernel)

int q4_dims(const htm_q4_shape* s, const char* who, Q4Dims* d) {
    if (!s) return htm_fail(HTM_E_INVALID, "%s: null shape", who);
    if (s->n_models < 1 || s->n_inputs < 1 || s->n_inputs > Q4_MAX_INPUTS || s->n_heads < 1 || s->n_heads > 64 ||
        s->n_outputs < 1 || s->n_outputs > 65536)
        return htm_fail(HTM_E_INVALID, "%s: shape out of range (models >= 1, inputs 1..65536, heads 1..64, outputs 1..65536)", who);
    if (s->group != 32 && s->group != 64 && s->group != 128)
        return htm_fail(HTM_E_INVALID, "%s: group must be 32, 64 or 128", who);
    d->nm = s->n_models;
    d->ni = s->n_inputs;
    d->nh = s->n_heads;
    d->no = s->n_outputs;
    d->group = s->group;
    d->nblk = (s->n_outputs + Q4_BLK - 1) / Q4_BLK;
    d->ngrp = (d->nblk * Q4_BLK + s->group - 1) / s->group;
    if ((int64_t)d->nh * d->nblk * Q4_BLK > 1048576)
        return htm_fail(HTM_E_INVALID, "%s: n_heads * padded outputs must be <= 1048576", who);
    d->scales = (uint32_t)(d->nh * d->nblk) * 16u;
    d->pitch = (d->scales + 2u * (uint32_t)(d->nh * d->ngrp) + 63u) / 64u * 64u;
    return HTM_OK;
}

__device__ __forceinline__ float bf16_up(uint32_t h) { return __uint_as_float(h << 16); }

// float32 -> bfloat16 to nearest even (finite values)
__device__ __forceinline__ uint32_t bf16_round(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

__device__ __forceinline__ float x_up(float v) { return v; }
__device__ __forceinline__ float x_up(__half v) { return __half2float(v); }
__device__ __forceinline__ float x_up(__hip_bfloat16 v) { return __bfloat162float(v); }

// ---------------------------------------------------------------- quantiser
// One workgroup per record, 16 lanes per group: a lane holds neighbouring pairs of
// its weights, a byte of codes each, so that weights and codes go by whole lines.
// 2 x 24,576 x 7 x 480: float64 483 us (2.9 TB/s), float32 452 us, which the
// divisions bound (a group a thread, whose reads and writes share no line: 5.1 and
// 6.0 ms).
template <typename T>
__global__ void __launch_bounds__(Q4_NT) q4_quantise_kernel(Q4Dims d, const T* __restrict__ w, int64_t ms, int64_t is,
                                                            int64_t hs, uint8_t* __restrict__ rec, int32_t* bad) {
    const int64_t rows = (int64_t)d.nm * d.ni;
    const int per = d.nh * d.ngrp, lane = threadIdx.x & 15, padded = d.nblk * Q4_BLK;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t model = row / d.ni;
        const T* in = w + model * ms + (row - model * d.ni) * is;
        uint8_t* r = rec + row * (int64_t)d.pitch;
        for (int k = threadIdx.x >> 4; k < per; k += Q4_NT / 16) {
            const int h = k / d.ngrp, g = k - h * d.ngrp, o0 = g * d.group + 2 * lane;
            const T* src = in + (int64_t)h * hs;
            T v[4][2];
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int j = 0; j < 2; j++) v[q][j] = q * 32 < d.group && o0 + q * 32 + j < d.no ? src[o0 + q * 32 + j] : (T)0;
            double amax = 0.0;
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const double a = fabs((double)v[q][j]);
                    amax = a <= 7.0 * Q4_MAX_SCALE ? fmax(amax, a) : INFINITY;  // (NaN among them)
                }
#pragma unroll
            for (int m = 8; m; m >>= 1) amax = fmax(amax, __shfl_xor(amax, m));
            const bool odd = amax == INFINITY;
            const float s0 = (float)(amax / 7.0);
            const uint32_t sb = (double)s0 >= Q4_MIN_SCALE && !odd ? bf16_round(s0) : 0u;
            const double s = (double)bf16_up(sb);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int o = o0 + q * 32;
                if (q * 32 >= d.group || o >= padded) break;
                uint32_t c[2];
#pragma unroll
                for (int j = 0; j < 2; j++)
                    c[j] = sb ? (uint32_t)(8 + (int)fmin(fmax(rint((double)v[q][j] / s), -7.0), 7.0)) : 8u;
                r[((uint32_t)(h * padded) + o) >> 1] = (uint8_t)(c[0] | (c[1] << 4));
            }
            if (lane == 0) {
                reinterpret_cast<uint16_t*>(r + d.scales)[k] = (uint16_t)sb;
                if (odd) *bad = 1;
            }
        }
    }
}

int q4_quantise_launch(const Q4Dims& d, const void* w, int32_t dtype, int64_t ms, int64_t is, int64_t hs, void* rec,
                       int32_t* bad, hipStream_t st) {
    const int64_t rows = (int64_t)d.nm * d.ni;
    const dim3 grid((uint32_t)(rows < 65536 ? rows : 65536));
    if (dtype == HTM_T_F64)
        hipLaunchKernelGGL(q4_quantise_kernel<double>, grid, dim3(Q4_NT), 0, st, d, (const double*)w, ms, is, hs,
                           (uint8_t*)rec, bad);
    else
        hipLaunchKernelGGL(q4_quantise_kernel<float>, grid, dim3(Q4_NT), 0, st, d, (const float*)w, ms, is, hs,
                           (uint8_t*)rec, bad);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 quantise launch failed");
}

// *bad = 1 if a record's scale is neither 0 nor within its range: a thread per scale, neighbours side by side.  256 x
// 24,576 records of 105 scales: 0.6 ms.
__global__ void __launch_bounds__(Q4_NT) q4_check_kernel(Q4Dims d, const uint8_t* __restrict__ rec, int32_t* bad) {
    const int per = d.nh * d.ngrp;
    const int64_t total = (int64_t)d.nm * d.ni * per;
    bool odd = false;
    for (int64_t i = (int64_t)blockIdx.x * Q4_NT + threadIdx.x; i < total; i += (int64_t)gridDim.x * Q4_NT) {
        const int64_t row = i / per;
        const uint16_t b = reinterpret_cast<const uint16_t*>(rec + row * d.pitch + d.scales)[i - row * per] & 0x7FFFu;
        odd |= b && (b < (uint16_t)((127 - 110) << 7) || b > (uint16_t)((127 + 100) << 7));
    }
    if (odd) *bad = 1;
}

// ------------------------------------------------------------------ products
// A record's block: 32 outputs' codes in 16 bytes, under one scale.  A code's four
// bits are masked where they lie, under the exponent that makes the lowest of them
// count one, and a subtraction leaves code - 8, exactly: a weight takes part as the
// number it stands for (11 bits at most), so that one of zero adds nothing, however
// large its scale.  Three full-rate instructions a weight, and a shift for eight.
// Measured, us (4,096 rows of 600 of 24,576 inputs, 480 outputs; 256 rows of own
// matrices, 7 heads): 108 and 83; by pairs of half floats, a packed subtraction and
// mixed FMAs 115 and 92; by v_cvt_off_f32_i4 124 and 98.  (Sums of scale * code with 8 *
// the sum of scales taken off at the end take 95 and 78, but a large scale then rounds
// the other inputs' weights away.)
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ half2_t as_half2(uint32_t u) { return __builtin_bit_cast(half2_t, u); }

// (a & mask) | bits as one instruction: its operands allow one constant, so the
// other has to be kept in a register, which the compiler does not do by itself.
__device__ __forceinline__ uint32_t in_vgpr(uint32_t c) {
    asm("" : "+v"(c));
    return c;
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) { return (a & mask) | bits; }

struct Q4Acc {
    float v[Q4_BLK];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < Q4_BLK; j++) v[j] = 0.0f;
    }
    // + m * (codes - 8), m the scale
    __device__ __forceinline__ void add(uint4 c, float m) {
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        uint32_t e[5];  // 2^(23 - 4 n): bits 4 n and up count ones
#pragma unroll
        for (int n = 0; n < 5; n++) e[n] = in_vgpr((uint32_t)(127 + 23 - 4 * n) << 23);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t h = w[k] >> 12;
            float* p = v + k * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int n = j < 5 ? j : j - 3;
                const float x = __uint_as_float(and_or(j < 5 ? w[k] : h, 0xFu << (4 * n), e[n]));
                p[j] = __builtin_fmaf(x - ((float)(1u << (23 - 4 * n)) + 8.0f), m, p[j]);
            }
        }
    }
};

// The workgroup's threads are slots x blocks: thread (slot, block) has summed
// its share of the inputs for one block's 32 outputs.  Sums over the slots, in
// a fixed order, through LDS (16 of the 32 at a time, rows of nt + 1 floats);
// put(output, y) is called once for each of the workgroup's nblk * 32 outputs.
template <typename PUT>
__device__ __forceinline__ void q4_join(Q4Acc& a, int nblk, int slots, float* sm, PUT put) {
    const int nt = blockDim.x, nout = nblk * 16;
    const int parts = nout < nt ? nt / nout : 1;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 16; j++) sm[j * (nt + 1) + threadIdx.x] = a.v[half * 16 + j];
        __syncthreads();
        if (parts == 1) {
            for (int o = threadIdx.x; o < nout; o += nt) {
                const float* p = sm + (o & 15) * (nt + 1) + (o >> 4);
                float y = 0.0f;
                for (int s = 0; s < slots; s++) y += p[s * nblk];
                put((o >> 4) * Q4_BLK + half * 16 + (o & 15), y);
            }
        } else {  // few outputs: several threads each take a run of slots, then one adds up theirs
            const int part = threadIdx.x / nout, o = threadIdx.x - part * nout;
            const int each = (slots + parts - 1) / parts;
            const float* p = sm + (o & 15) * (nt + 1) + (o >> 4);
            float y = 0.0f;
            if (part < parts)
                for (int s = part * each; s < min(slots, part * each + each); s++) y += p[s * nblk];
            __syncthreads();
            if (part < parts) sm[threadIdx.x] = y;
            __syncthreads();
            if (threadIdx.x < (uint32_t)nout) {
                y = 0.0f;
                for (int k = 0; k < parts; k++) y += sm[k * nout + o];
                put((o >> 4) * Q4_BLK + half * 16 + (o & 15), y);
            }
        }
    }
}

// softmax of y[0..nl) to q[0..no), zero behind nl, by one wave (y == q is fine)
__device__ __forceinline__ void q4_wave_softmax(const float* y, float* q, int nl, int no, int lane) {
    float m = -INFINITY, t = 0.0f, v[Q4_MAX_SOFTMAX / 64];
#pragma unroll
    for (int j = 0; j < Q4_MAX_SOFTMAX / 64; j++) {
        const int k = j * 64 + lane;
        v[j] = k < nl ? y[k] : -INFINITY;
        m = fmaxf(m, v[j]);
    }
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
#pragma unroll
    for (int j = 0; j < Q4_MAX_SOFTMAX / 64; j++) {
        v[j] = j * 64 + lane < nl ? expf(v[j] - m) : 0.0f;
        t += v[j];
    }
    for (int k = 32; k; k >>= 1) t += __shfl_xor(t, k);
#pragma unroll
    for (int j = 0; j < Q4_MAX_SOFTMAX / 64; j++)
        if (j * 64 + lane < no) q[j * 64 + lane] = j * 64 + lane < nl ? v[j] / t : 0.0f;
}

#define Q4_LIST 2048   // active inputs listed at a time
#define Q4_WORDS 8     // pattern words of a thread (65,536 inputs by 256 threads)

// Word bitmaps.  One workgroup per (row, run of cblk blocks of the record, which
// may span heads).  The active inputs are listed in LDS in ascending order:
// the words that are not empty are compacted first and then listed by two
// threads each, since a bursting column sets a word's bits together.  Each slot takes
// an even share of the list, its threads the run's blocks side by side, so that
// a record is read in one piece.  SOFTMAX: the run is whole heads, whose
// probabilities are written instead.
//
// One row is its chain of latencies: pattern, list, records, join, 7 us of 420
// waves for 1.2 MB.  Rows that share a matrix find it in the caches and are bound by
// instructions: 4,096 rows of 768 columns x 32 cells, some 600 of them active, 480
// outputs, are 7.2e7 wave instructions (3.9 a weight, of which mask, subtraction,
// FMA and shift 3.1), 75 us of issue at 2.5 cycles each, in 108 us; of 2,048 x 12, 280
// active, 58 us.  Rows of their own matrices (256 rows, 7 x 480 outputs, 295 MB in 83
// us; of 2,048 x 12 37) are bound by what one workgroup moves and unpacks: the 40 % of
// the rows whose columns burst, 1,280 cells each, hold 85 % of the bytes, and some 100
// workgroups work on while the others have ended.
template <bool SOFTMAX>
__global__ void __launch_bounds__(1024) q4_rows_kernel(Q4Dims d, const uint8_t* __restrict__ rec,
                                                       const uint32_t* __restrict__ pat, int64_t ps, int per_model,
                                                       int row0, int cblk, const int32_t* __restrict__ live,
                                                       float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) uint32_t list[Q4_LIST];  // record offsets / 64
    __shared__ uint32_t wsum[16];
    extern __shared__ __attribute__((aligned(16))) float sm[];       // compacted words, then the join's rows
    const int nt = blockDim.x, nwave = nt >> 6;
    const int row = row0 + blockIdx.y, b0 = blockIdx.x * cblk;
    const int nblk = min(cblk, d.nh * d.nblk - b0);
    const int slots = nt / nblk;
    const int slot = threadIdx.x / nblk, blk = b0 + threadIdx.x - slot * nblk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t* p = pat + (int64_t)row * ps;
    const int words = d.ni / 32;

    // the thread's words: how many are not empty, and their bits
    const int each = (words + nt - 1) / nt, w0 = threadIdx.x * each;
    uint32_t x[Q4_WORDS], mine = 0;
#pragma unroll
    for (int k = 0; k < Q4_WORDS; k++) {
        x[k] = k < each && w0 + k < words ? p[w0 + k] : 0u;
        mine += __popc(x[k]) + (x[k] ? 1u << 18 : 0u);  // (at most 65,536 bits of 2,048 words)
    }
    uint32_t at = mine;
    for (int k = 1; k < 64; k <<= 1) {
        const uint32_t o = __shfl_up(at, k);
        if (lane >= k) at += o;
    }
    if (lane == 63) wsum[wave] = at;
    __syncthreads();
    uint32_t all = 0;
    at -= mine;
    for (int k = 0; k < nwave; k++) {
        const uint32_t s = wsum[k];
        if (k < wave) at += s;
        all += s;
    }
    const uint32_t n = all & 0x3FFFFu, full = all >> 18;
    uint2* cw = reinterpret_cast<uint2*>(sm);
#pragma unroll
    for (int k = 0; k < Q4_WORDS; k++)
        if (x[k]) {
            cw[at >> 18] = make_uint2(x[k], ((uint32_t)(w0 + k) << 17) | (at & 0x3FFFFu));  // (a word begins below 65,536)
            at += __popc(x[k]) + (1u << 18);
        }
    __syncthreads();

    Q4Acc acc;
    acc.clear();
    const int h = blk / d.nblk;
    const uint8_t* base = rec + (int64_t)(row / per_model) * d.ni * d.pitch;
    const uint8_t* cb = base + blk * 16;
    const uint8_t* sb = base + d.scales + 2 * (h * d.ngrp + (blk - h * d.nblk) * Q4_BLK / d.group);
    const uint32_t pitch64 = d.pitch / 64;
    for (uint32_t r0 = 0; r0 < n; r0 += Q4_LIST) {  // (a second round only beyond Q4_LIST active inputs)
        if (r0) __syncthreads();
        for (uint32_t j = threadIdx.x >> 1; j < full; j += nt >> 1) {
            const uint2 v = cw[j];
            const uint32_t lo = v.x & 0xFFFFu;
            uint32_t b = threadIdx.x & 1 ? v.x & 0xFFFF0000u : lo;
            uint32_t q = (v.y & 0x1FFFFu) + (threadIdx.x & 1 ? __popc(lo) : 0) - r0;
            const uint32_t first = (v.y >> 17) * 32u - 1u;
            for (; b; b &= b - 1, q++)
                if (q < Q4_LIST) list[q] = (first + __ffs(b)) * pitch64;
        }
        __syncthreads();
        const int m = (int)min(n - r0, (uint32_t)Q4_LIST);
        if (slot < slots) {
            // every slot's share, and one more for the first m % slots of them
            const int share = m / slots, more = m - share * slots;
            int i = slot * share + min(slot, more);
            auto some = [&](auto count) {
                constexpr int U = decltype(count)::value;
                uint4 c[U];
                uint32_t s[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint64_t r = (uint64_t)list[i + u] << 6;
                    c[u] = *reinterpret_cast<const uint4*>(cb + r);
                    s[u] = *reinterpret_cast<const uint16_t*>(sb + r);
                }
                __builtin_amdgcn_sched_barrier(0);  // (every load is under way before the first is waited for)
#pragma unroll
                for (int u = 0; u < U; u++) acc.add(c[u], bf16_up(s[u]));
                i += U;
            };
            for (int k = share; k >= 4; k -= 4) some(std::integral_constant<int, 4>());
            if (share & 2) some(std::integral_constant<int, 2>());
            if (share & 1) some(std::integral_constant<int, 1>());
            if (slot < more) some(std::integral_constant<int, 1>());
        }
    }
    float* o = out + (int64_t)row * d.nh * d.no;
    if (!SOFTMAX) {
        q4_join(acc, nblk, slots, sm, [&](int k, float y) {
            const int b = b0 + (k >> 5), hh = b / d.nblk, j = (b - hh * d.nblk) * Q4_BLK + (k & 31);
            if (j < d.no) o[hh * d.no + j] = y;
        });
        return;
    }
    float* y_sh = sm + 16 * (nt + 1);
    q4_join(acc, nblk, slots, sm, [&](int k, float y) { y_sh[k] = y; });
    __syncthreads();
    // a wave per head
    int nl = d.no;
    if (live) nl = min(max(live[row / per_model], 0), d.no);
    const int stride = d.nblk * Q4_BLK;
    for (int hh = wave; hh < nblk / d.nblk; hh += nwave)
        q4_wave_softmax(y_sh + hh * stride, o + (b0 / d.nblk + hh) * d.no, nl, d.no, lane);
}

// The softmax alone, in place: a wave per (row, head); 64 rows of 1,000 4 us, one
// wave's chain, behind products of 15 us.
__global__ void __launch_bounds__(Q4_NT) q4_softmax_kernel(Q4Dims d, const int32_t* __restrict__ live, int per_model,
                                                           int64_t total, float* __restrict__ y) {
    const int64_t k = (int64_t)blockIdx.x * (Q4_NT / 64) + (threadIdx.x >> 6);
    if (k >= total) return;
    int nl = d.no;
    if (live) nl = min(max(live[k / d.nh / per_model], 0), d.no);
    q4_wave_softmax(y + k * d.no, y + k * d.no, nl, d.no, threadIdx.x & 63);
}

// Vectors of numbers.  One workgroup per (NX rows of one matrix, run of cb
// half blocks, range of inputs): the inputs of a tile that are not zero in
// every row are listed in LDS with the rows' numbers, the slots share the list
// evenly, and a thread keeps its half block's 16 outputs of all NX rows, so that
// a weight is read and unpacked once for all of them.  Here a code's bits get the
// exponent under which they count ones (1024 + code, or 64 + code), and a packed
// subtraction leaves code - 8, exactly: a weight takes part as the number it
// stands for.  2,048 column confidences, 6 % of them not zero, to 480: 5.5 us, one
// workgroup's chain; 24,576 numbers to 7 x 480: 22 us for 47 MB, of which the weights'
// 4.2 instructions are half.
#define MV_NT 256
#define MV_HB 16     // outputs of a half block

template <int NX>
struct MvAcc {
    float v[NX][MV_HB];
    __device__ __forceinline__ void add(uint2 c, float s, const float* x, uint32_t e1032, uint32_t e72) {
        const half2_t k0 = {(_Float16)1032.0f, (_Float16)1032.0f}, k1 = {(_Float16)72.0f, (_Float16)72.0f};
        const uint32_t w[2] = {c.x, c.y};
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t h = w[k] >> 8;
            const half2_t q[4] = {as_half2(and_or(w[k], 0x000F000Fu, e1032)) - k0, as_half2(and_or(w[k], 0x00F000F0u, e72)) - k1,
                                  as_half2(and_or(h, 0x000F000Fu, e1032)) - k0, as_half2(and_or(h, 0x00F000F0u, e72)) - k1};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // (the weight first, exactly: scale * x may overflow or vanish where the weight's product does not)
                const float y = __builtin_fmaf((float)(j < 4 ? q[j & 3].x : q[j & 3].y), s, 0.0f);
#pragma unroll
                for (int r = 0; r < NX; r++) v[r][k * 8 + j] = __builtin_fmaf(x[r], y, v[r][k * 8 + j]);
            }
        }
    }
};

template <typename T, int NX>
__global__ void __launch_bounds__(MV_NT, NX == 4 ? 3 : 4)
    q4_matvec_kernel(Q4Dims d, const uint8_t* __restrict__ rec, const T* __restrict__ x, int64_t xs, int per, int y0,
                     int passes, int cb, int chunks, int range, float* __restrict__ out, int64_t split_stride) {
    constexpr int KPT = 8 / NX, TILE = MV_NT * KPT;  // inputs of a thread and of a tile
    __shared__ uint32_t list[TILE];
    __shared__ __attribute__((aligned(16))) float xv[TILE][NX];
    __shared__ uint32_t wsum[MV_NT / 64];
    __shared__ float sm[MV_HB][MV_NT + 1];
    __shared__ float sums[MV_NT];
    const int splits = gridDim.x / chunks, split = blockIdx.x % splits, chunk = blockIdx.x / splits;
    const int y = y0 + blockIdx.y, model = y / passes, q0 = (y - model * passes) * NX;
    const int nx = min(NX, per - q0);
    const int64_t row = (int64_t)model * per + q0;
    const int halves = d.nh * d.nblk * 2, b0 = chunk * cb, nb = min(cb, halves - b0);
    const int slots = MV_NT / nb, slot = threadIdx.x / nb, hb = b0 + threadIdx.x - slot * nb;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint8_t* base = rec + (int64_t)model * d.ni * d.pitch;
    const int h = hb / (d.nblk * 2);
    const uint8_t* cbase = base + hb * 8;
    const uint8_t* sbase = base + d.scales + 2 * (h * d.ngrp + (hb - h * d.nblk * 2) * MV_HB / d.group);
    const uint32_t pitch64 = d.pitch / 64;
    const int k0 = split * range, k1 = min(d.ni, k0 + range);
    const uint32_t e1032 = in_vgpr(0x64006400u), e72 = in_vgpr(0x54005400u);
    MvAcc<NX> a;
#pragma unroll
    for (int r = 0; r < NX; r++)
#pragma unroll
        for (int j = 0; j < MV_HB; j++) a.v[r][j] = 0.0f;
    T next[KPT][NX];  // inputs t0 + i * MV_NT + thread; as they are: a conversion would wait for them
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            const int k = t0 + i * MV_NT + (int)threadIdx.x;
#pragma unroll
            for (int r = 0; r < NX; r++) next[i][r] = k < k1 && r < nx ? x[(row + r) * xs + k] : T(0.0f);
        }
    };
    fetch(k0);
    for (int t0 = k0; t0 < k1; t0 += TILE) {
        uint64_t bal[KPT];
        uint32_t cnt = 0;
        float mine[KPT][NX];
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            bool some = false;
#pragma unroll
            for (int r = 0; r < NX; r++) {
                mine[i][r] = x_up(next[i][r]);
                some |= mine[i][r] != 0.0f;
            }
            bal[i] = __ballot(some);
            cnt += (uint32_t)__popcll(bal[i]);
        }
        if (lane == 0) wsum[wave] = cnt;
        __syncthreads();
        uint32_t at = 0, m = 0;
#pragma unroll
        for (int k = 0; k < MV_NT / 64; k++) {
            if (k < wave) at += wsum[k];
            m += wsum[k];
        }
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            if ((bal[i] >> lane) & 1) {
                const uint32_t q = at + (uint32_t)__popcll(bal[i] & ((1ull << lane) - 1ull));
                list[q] = (uint32_t)(t0 + i * MV_NT + (int)threadIdx.x) * pitch64;
#pragma unroll
                for (int r = 0; r < NX; r++) xv[q][r] = mine[i][r];
            }
            at += (uint32_t)__popcll(bal[i]);
        }
        __syncthreads();
        fetch(t0 + TILE);  // (the next tile's numbers meanwhile)
        if (slot < slots) {
            const int share = (int)m / slots, more = (int)m - share * slots;
            int i = slot * share + min(slot, more);
            auto step = [&](auto count) {
                constexpr int U = decltype(count)::value;
                uint2 c[U];
                uint32_t s[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint64_t r = (uint64_t)list[i + u] << 6;
                    c[u] = *reinterpret_cast<const uint2*>(cbase + r);
                    s[u] = *reinterpret_cast<const uint16_t*>(sbase + r);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float xr[NX];
#pragma unroll
                    for (int r = 0; r < NX; r++) xr[r] = xv[i + u][r];
                    a.add(c[u], bf16_up(s[u]), xr, e1032, e72);
                }
                i += U;
            };
            int k = share;
            for (; k >= 8; k -= 8) step(std::integral_constant<int, 8>());
            if (k & 4) step(std::integral_constant<int, 4>());
            if (k & 2) step(std::integral_constant<int, 2>());
            if (k & 1) step(std::integral_constant<int, 1>());
            if (slot < more) step(std::integral_constant<int, 1>());
        }
    }
    float* o = out + split * split_stride + row * d.nh * d.no;
    const int nout = nb * MV_HB;
    const auto put = [&](int r, int k, float y) {
        const int b = b0 + (k >> 4), hh = b / (d.nblk * 2), j = (b - hh * d.nblk * 2) * MV_HB + (k & 15);
        if (j < d.no) o[(int64_t)r * d.nh * d.no + hh * d.no + j] = y;
    };
    // (few outputs: several threads each take a run of slots, then one adds up theirs)
    const int parts = max(MV_NT / nout, 1), each = (slots + parts - 1) / parts;
    const int part = threadIdx.x / nout, out0 = threadIdx.x - part * nout;
#pragma unroll
    for (int r = 0; r < NX; r++) {
        if (r >= nx) break;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < MV_HB; j++) sm[j][threadIdx.x] = a.v[r][j];
        __syncthreads();
        if (parts == 1) {
            for (int k = threadIdx.x; k < nout; k += MV_NT) {
                const float* p = &sm[k & 15][k >> 4];
                float y = 0.0f;
                for (int s = 0; s < slots; s++) y += p[s * nb];
                put(r, k, y);
            }
        } else {
            const float* p = &sm[out0 & 15][out0 >> 4];
            float y = 0.0f;
            if (part < parts)
                for (int s = part * each; s < min(slots, part * each + each); s++) y += p[s * nb];
            sums[threadIdx.x] = y;
            __syncthreads();
            if ((int)threadIdx.x < nout) {
                for (int k = 1; k < parts; k++) y += sums[k * nout + threadIdx.x];
                put(r, threadIdx.x, y);
            }
        }
    }
}

// Several rows at once, by matrix instructions.  v_mfma_f32_16x16x32_bf16 takes 16
// rows' numbers for 32 inputs (A) and those inputs' weights of 16 outputs (B).  A
// weight scale * (code - 8) has up to 11 bits, too many for a bfloat16 (a float16 would
// hold them, but not the range of all scales): the scale's
// upper and lower four bits make two bfloat16 products that are exact, and a
// number takes one (bfloat16), two (float16) or three (float32) bfloat16 parts,
// so that every product in the sum is exact and only float32 sums round, as in the
// kernel above, while a weight costs some 4.4 instructions for all 16 rows
// instead of 3 and one for each row.  Matrix instructions take what lies below
// float32's normal numbers as zero: scales are kept off that range, and of x and the
// products 2^-126 may be lost.
//
// One workgroup per (16 rows of one matrix, 16 half blocks, range of inputs).  A wave
// takes every fourth 64 inputs of the range for itself: those that are not zero in
// every row are listed in a ring in LDS with their numbers' parts, and whenever the
// ring holds 32, they are a step: lane l loads inputs (l / 16) * 8 .. + 7 of half block
// l % 16, which are B for each of the half block's 16 outputs: 16 sums of [16 rows x
// 16 half blocks], one for each output of a half block.
//
// 8 rows of 24,576 bfloat16 to 7 x 480: 25 us and 5 us for the join (47 MB: 10 us),
// bound by instructions: 8.2e6 of a wave, 4.6 a weight and lane, at the 5 cycles each
// that one or two waves a SIMD reach, are 18 us, the matrix instructions 3, the first
// records and the waves' join the rest.  A list for the whole workgroup, with barriers:
// 31 us; registers for three waves a SIMD spill: 47.  A wave's next numbers are read
// while it works; kept as they are, since a conversion waits for them at once: 30 us.
#define MM_NT 256
#define MM_ROWS 16
#define MM_RING 64               // listed inputs of a wave: less than 32 left over and 32 new ones
#define MM_PITCH (MM_RING + 8)   // bfloat16 of a row in LDS: 16-byte reads of 16 rows fall on different banks
#define MM_COLS 272              // floats of a row in the join: 16 x 17

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct MmParts { static constexpr int n = 3; };
template <> struct MmParts<__half> { static constexpr int n = 2; };
template <> struct MmParts<__hip_bfloat16> { static constexpr int n = 1; };

// LDS that a wave's lanes write for each other: in order for the compiler too
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ f32x4 mm(bf16x8 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T>
__global__ void __launch_bounds__(MM_NT, 2)
    q4_mfma_kernel(Q4Dims d, const uint8_t* __restrict__ rec, const T* __restrict__ x, int64_t xs, int per, int y0,
                   int passes, int tiles, int range, float* __restrict__ out, int64_t split_stride) {
    constexpr int P = MmParts<T>::n;
    extern __shared__ __attribute__((aligned(16))) uint8_t mm_sh[];
    __shared__ uint32_t lists[MM_NT / 64][MM_RING];
    const int splits = gridDim.x / tiles, split = blockIdx.x % splits, tile = blockIdx.x / splits;
    const int y = y0 + blockIdx.y, model = y / passes, q0 = (y - model * passes) * MM_ROWS;
    const int nx = min(MM_ROWS, per - q0);
    const int64_t row = (int64_t)model * per + q0;
    const int halves = d.nh * d.nblk * 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint16_t* xa = reinterpret_cast<uint16_t*>(mm_sh) + wave * (P * MM_ROWS * MM_PITCH);  // [P][MM_ROWS][MM_PITCH]
    uint32_t* list = lists[wave];
    const int hb = min(tile * 16 + (lane & 15), halves - 1);  // (behind the last: computed again and not written)
    const uint8_t* base = rec + (int64_t)model * d.ni * d.pitch;
    const int h = hb / (d.nblk * 2);
    const uint8_t* cbase = base + hb * 8;
    const uint8_t* sbase = base + d.scales + 2 * (h * d.ngrp + (hb - h * d.nblk * 2) * MV_HB / d.group);
    const uint32_t pitch64 = d.pitch / 64;
    const int k0 = split * range, k1 = min(d.ni, k0 + range);
    const uint32_t e1032 = in_vgpr(0x64006400u), e72 = in_vgpr(0x54005400u);
    f32x4 acc[MV_HB];
#pragma unroll
    for (int j = 0; j < MV_HB; j++) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    T next[MM_ROWS / 2];  // of input lane % 32, rows r0 .. + 7; as they are: a conversion would wait for them
    const int r0 = (lane >> 5) * (MM_ROWS / 2), nr = nx - r0;
    const T* xr = x + (row + r0) * xs + (lane & 31);
    auto fetch = [&](int t) {
        const bool in = t + (lane & 31) < k1;
#pragma unroll
        for (int r = 0; r < MM_ROWS / 2; r++) next[r] = in && r < nr ? xr[r * xs + t] : T(0.0f);
    };
    int head = 0, have = 0;  // the ring's first listed input and how many there are
    bool wild = false;       // an infinity or a NaN among them, or before
    const auto step = [&](int q) {
        const int q8 = q + (lane >> 4) * 8;
        uint2 c[8];
        uint32_t sc[8];
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const uint64_t o = (uint64_t)list[q8 + r] << 6;
            c[r] = *reinterpret_cast<const uint2*>(cbase + o);
            sc[r] = *reinterpret_cast<const uint16_t*>(sbase + o);
        }
        bf16x8 a[P];
#pragma unroll
        for (int p = 0; p < P; p++)
            a[p] = *reinterpret_cast<const bf16x8*>(xa + (p * MM_ROWS + (lane & 15)) * MM_PITCH + q8);
        __builtin_amdgcn_sched_barrier(0);  // (every load is under way before the first is waited for)
        // (the scale's lower part may be zero where the weight is not: infinity meets the upper one alone)
        u32x4 fin = __builtin_bit_cast(u32x4, a[0]);
        if (wild) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if ((fin[k] & 0x7F80u) == 0x7F80u) fin[k] &= 0xFFFF0000u;
                if ((fin[k] & 0x7F800000u) == 0x7F800000u) fin[k] &= 0x0000FFFFu;
            }
        }
        const bf16x8 a0 = __builtin_bit_cast(bf16x8, fin);
        float hi[8], lo[8];
#pragma unroll
        for (int r = 0; r < 8; r++) {
            hi[r] = bf16_up(sc[r] & 0xFFF0u);
            lo[r] = bf16_up(sc[r]) - hi[r];
        }
#pragma unroll
        for (int g = 0; g < 4; g++) {  // four outputs: half a word of each input's codes
            uint32_t w[4];
#pragma unroll
            for (int p = 0; p < 4; p++)
                w[p] = __builtin_amdgcn_perm(g < 2 ? c[2 * p + 1].x : c[2 * p + 1].y, g < 2 ? c[2 * p].x : c[2 * p].y,
                                             g & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const half2_t bias = n & 1 ? half2_t{(_Float16)72.0f, (_Float16)72.0f}
                                           : half2_t{(_Float16)1032.0f, (_Float16)1032.0f};
                u32x4 bh, bl;
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const uint32_t u = n < 2 ? w[p] : w[p] >> 8;
                    const half2_t q2 = as_half2(n & 1 ? and_or(u, 0x00F000F0u, e72) : and_or(u, 0x000F000Fu, e1032)) - bias;
                    const float h0 = __builtin_fmaf((float)q2.x, hi[2 * p], 0.0f);
                    const float h1 = __builtin_fmaf((float)q2.y, hi[2 * p + 1], 0.0f);
                    const float l0 = __builtin_fmaf((float)q2.x, lo[2 * p], 0.0f);
                    const float l1 = __builtin_fmaf((float)q2.y, lo[2 * p + 1], 0.0f);
                    bh[p] = __builtin_amdgcn_perm(__float_as_uint(h1), __float_as_uint(h0), 0x07060302u);
                    bl[p] = __builtin_amdgcn_perm(__float_as_uint(l1), __float_as_uint(l0), 0x07060302u);
                }
                const int j = g * 4 + n;
#pragma unroll
                for (int p = 0; p < P; p++) {
                    acc[j] = mm(p ? a[p] : a0, bl, acc[j]);
                    acc[j] = mm(a[p], bh, acc[j]);
                }
            }
        }
    };
    fetch(k0 + wave * 32);
    for (int t = k0 + wave * 32; t < k1; t += MM_NT / 2) {
        bool some = false, odd = false;
        float mine[MM_ROWS / 2];
#pragma unroll
        for (int r = 0; r < MM_ROWS / 2; r++) {
            mine[r] = x_up(next[r]);
            some |= mine[r] != 0.0f;
            odd |= !(fabsf(mine[r]) < INFINITY);
        }
        const uint64_t both = __ballot(some);
        const uint32_t bal = (uint32_t)both | (uint32_t)(both >> 32);
        wild |= __ballot(odd) != 0;
        const int at = (head + have + __popc(bal & ((1u << (lane & 31)) - 1u))) & (MM_RING - 1);
        if ((bal >> (lane & 31)) & 1) {
            list[at] = (uint32_t)(t + (lane & 31)) * pitch64;
            uint16_t* to = xa + r0 * MM_PITCH + at;
#pragma unroll
            for (int r = 0; r < MM_ROWS / 2; r++) {
                if (r >= nr) break;  // (what the missing rows' lanes read is their own rows' affair, and not written)
                float v = mine[r];
#pragma unroll
                for (int p = 0; p < P; p++) {
                    uint32_t u = __float_as_uint(v) & 0xFFFF0000u;
                    if (v != v) u = 0x7FC00000u;
                    // (what is left of an infinity or a NaN is not a part)
                    v = fabsf(v) < INFINITY ? v - __uint_as_float(u) : 0.0f;
                    to[(p * MM_ROWS + r) * MM_PITCH] = (uint16_t)(u >> 16);
                }
            }
        }
        have += __popc(bal);
        fetch(t + MM_NT / 2);  // (the next numbers meanwhile)
        wave_lds();
        if (have >= 32) {
            step(head);
            head ^= 32;
            have -= 32;
        }
        wave_lds();
    }
    if (have) {  // up to 32 behind the list: the range's first input, times zero
        if (lane >= have && lane < 32) {
            list[head + lane] = (uint32_t)k0 * pitch64;
            for (int r = 0; r < P * MM_ROWS; r++) xa[r * MM_PITCH + head + lane] = 0;
        }
        wave_lds();
        step(head);
    }
    // the four waves' sums
    __syncthreads();
    float* jn = reinterpret_cast<float*>(mm_sh);  // [wave][row][output of 16][half block of 16 + 1]
#pragma unroll
    for (int j = 0; j < MV_HB; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane >> 4) * 4 + i;
            if (r < nx) jn[(wave * nx + r) * MM_COLS + j * 17 + (lane & 15)] = acc[j][i];
        }
    __syncthreads();
    const int b = tile * 16 + (int)threadIdx.x / 16, j = threadIdx.x & 15;
    const int hh = b / (d.nblk * 2), col = (b - hh * d.nblk * 2) * MV_HB + j;
    if (b >= halves || col >= d.no) return;
    float* o = out + split * split_stride + row * d.nh * d.no + hh * d.no + col;
    for (int r = 0; r < nx; r++) {
        const float* p = jn + r * MM_COLS + j * 17 + threadIdx.x / 16;
        const int w = nx * MM_COLS;
        o[(int64_t)r * d.nh * d.no] = (p[0] + p[w]) + (p[2 * w] + p[3 * w]);
    }
}

// The ranges' sums added up: 64 outputs a workgroup, a quarter of the ranges a
// wave, in a fixed order.  32 ranges of 8 x 7 x 480: 4.8 us, the latency of eight
// loads.
__global__ void __launch_bounds__(256) q4_join_kernel(const float* __restrict__ part, int splits, int64_t n,
                                                      float* __restrict__ out) {
    __shared__ float sm[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t k = (int64_t)blockIdx.x * 64 + lane;
    const int each = (splits + 3) / 4, s1 = min(splits, wave * each + each);
    float y = 0.0f;
    if (k < n) {
        int s = wave * each;
        for (; s + 8 <= s1; s += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = part[(s + j) * n + k];
#pragma unroll
            for (int j = 0; j < 8; j++) y += v[j];
        }
        for (; s < s1; s++) y += part[s * n + k];
    }
    sm[wave][lane] = y;
    __syncthreads();
    if (wave == 0 && k < n) out[k] = (sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]);
}

// rows checked against the matrices; *per = rows that share one
static int q4_rows(const Q4Dims& d, int32_t n_rows, const char* who, int* per) {
    if (n_rows < 0 || n_rows > 65535 * 32 || n_rows % d.nm)
        return htm_fail(HTM_E_INVALID, "%s: n_rows must be a multiple of n_models, at most 2097120", who);
    *per = n_rows / d.nm;
    return HTM_OK;
}

static int q4_aligned(const void* p, const char* who) {
    if (!p || (uintptr_t)p % 16) return htm_fail(HTM_E_INVALID, "%s: records must be 16-byte aligned", who);
    return HTM_OK;
}

extern "C" {

size_t htm_q4_record_bytes(const htm_q4_shape* s) {
    Q4Dims d;
    return q4_dims(s, __func__, &d) ? 0 : d.pitch;
}

int htm_q4_quantise(const htm_q4_shape* s, const void* w, int32_t dtype, int64_t ms, int64_t is, int64_t hs, void* rec,
                    int32_t* bad, void* stream) {
    Q4Dims d;
    if (int r = q4_dims(s, __func__, &d)) return r;
    if (int r = q4_aligned(rec, __func__)) return r;
    if (!w || !bad || (dtype != HTM_T_F32 && dtype != HTM_T_F64) || ms < 0 || is < 0 || hs < 0)
        return htm_fail(HTM_E_INVALID, "%s: invalid argument", __func__);
    return q4_quantise_launch(d, w, dtype, ms, is, hs, rec, bad, (hipStream_t)stream);
}

int htm_q4_check(const htm_q4_shape* s, const void* rec, int32_t* bad, void* stream) {
    Q4Dims d;
    if (int r = q4_dims(s, __func__, &d)) return r;
    if (int r = q4_aligned(rec, __func__)) return r;
    if (!bad) return htm_fail(HTM_E_INVALID, "%s: invalid argument", __func__);
    const int64_t blocks = ((int64_t)d.nm * d.ni * d.nh * d.ngrp + Q4_NT - 1) / Q4_NT;
    hipLaunchKernelGGL(q4_check_kernel, dim3((uint32_t)std::min<int64_t>(blocks, 16384)), dim3(Q4_NT), 0, (hipStream_t)stream, d,
                       (const uint8_t*)rec, bad);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 check launch failed");
}

static int q4_bitmap(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows,
                     const float* out, const char* who, Q4Dims* d, int* per) {
    if (int r = q4_dims(s, who, d)) return r;
    if (int r = q4_rows(*d, n_rows, who, per)) return r;
    if (d->ni % 32) return htm_fail(HTM_E_INVALID, "%s: patterns need n_inputs a multiple of 32", who);
    if (!n_rows) return HTM_OK;
    if (int r = q4_aligned(rec, who)) return r;
    if (!pat || !out || (n_rows > 1 && ps < d->ni / 32)) return htm_fail(HTM_E_INVALID, "%s: invalid argument", who);
    return HTM_OK;
}

}  // extern "C"

#define Q4_GRID_Y 65535  // rows of one launch

// More than 64 KiB of dynamic LDS: allowed once per kernel and device.
static int q4_raise_lds(const void* kernel, size_t lds, std::atomic<uint64_t>& raised) {
    if (lds <= 65536) return HTM_OK;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return htm_fail(HTM_E_HIP, "q4: no current device");
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (raised.load() & bit)) return HTM_OK;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 150 * 1024) != hipSuccess)
        return htm_fail(HTM_E_HIP, "q4: cannot raise the dynamic LDS limit to %zu B", lds);
    if (dev < 64) raised.fetch_or(bit);
    return HTM_OK;
}

// How a product is shared out: rows at a time, runs of half blocks and ranges of
// inputs, some 512 workgroups in all.  Measured, us, both launches:
//   rows, inputs, outputs          4 rows a pass   8 rows    matrix instructions
//   1, 24,576, 7 x 480             21 (one row)              32 (bfloat16 28)
//   4, 24,576, 7 x 480             29                        32 (bfloat16 28)
//   5, 24,576, 7 x 480                             43        32 (bfloat16 28)
//   8, 24,576, 7 x 480                             44        33 (bfloat16 28)
//   16, 24,576, 7 x 480                            76        35
//   8, 24,576, 480                                 16        14
//   12, 4,000, 7 x 480                             22        14
//   8, 24,576 with 6 % not zero, 7 x 480           14        18 (how many are zero is not known here)
// and for the first two columns, runs x ranges: 8, 24,576, 7 x 480: 7 x 73 44, 7 x
// 36 50, 4 x 64 58; 1, 4,000, 480: 2 x 16 9.3, 30 x 1 12.5.  In one launch while a
// tile holds the inputs (Python call included; in two it takes 12.4): 1, 2,048, 480 8.8;
// 2, 1,000, 480 8.5 (2, 2,048 11.6); 4, 500, 480 9.9 (4, 1,000 13.0); 8, 200, 480 10.1
// (8, 400 15.9).  Matrix instructions with ranges of 128 up to 4,096 inputs: 8, 4,000,
// 480 12.8, of 256 13.3.
struct MvPlan {
    bool mfma;
    int nx, passes, cb, chunks, splits, range;
};

static MvPlan mv_plan(const Q4Dims& d, int per) {
    MvPlan p;
    p.mfma = per >= 5;
    p.nx = p.mfma ? MM_ROWS : per >= 3 ? 4 : per;
    p.passes = (per + p.nx - 1) / p.nx;
    const int64_t y = (int64_t)d.nm * p.passes;
    const int halves = d.nh * d.nblk * 2;
    p.splits = 1;
    const int64_t few = 512;
    if (p.mfma) {
        const int64_t most = d.ni <= 256 ? 1 : (d.ni + (d.ni <= 4096 ? 127 : 255)) / (d.ni <= 4096 ? 128 : 256);
        p.chunks = (halves + 15) / 16;
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(few / (p.chunks * y), most));
        // (a range's workgroups on one XCD: their pieces of a record share its lines)
        if (p.splits >= 8) p.splits = p.splits / 8 * 8;
    } else if (d.ni <= MV_NT * 8 / p.nx && (halves + 3) / 4 * y <= few) {
        p.chunks = (halves + 3) / 4;
    } else {
        const int64_t most = (d.ni + 255) / 256;
        p.chunks = (halves + 15) / 16;
        if (p.chunks * most * y > few) p.chunks = (halves + 31) / 32;
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(few / (p.chunks * y), most));
    }
    p.cb = (halves + p.chunks - 1) / p.chunks;
    p.chunks = (halves + p.cb - 1) / p.cb;
    p.range = (d.ni + p.splits - 1) / p.splits;
    p.splits = (d.ni + p.range - 1) / p.range;
    return p;
}

template <typename T>
static int mv_launch(const MvPlan& p, const Q4Dims& d, const void* rec, const void* x, int64_t xs, int per, float* out,
                      int64_t stride, hipStream_t st) {
    const int64_t all = (int64_t)d.nm * p.passes;
    const size_t lds = std::max<size_t>((size_t)(MM_NT / 64) * MmParts<T>::n * MM_ROWS * MM_PITCH * 2,
                                        (size_t)4 * std::min(per, MM_ROWS) * MM_COLS * sizeof(float));
    static std::atomic<uint64_t> raised{0};
    if (p.mfma)
        if (int r = q4_raise_lds((const void*)q4_mfma_kernel<T>, lds, raised)) return r;
    for (int64_t y0 = 0; y0 < all; y0 += Q4_GRID_Y) {
        const dim3 grid(p.chunks * p.splits, (uint32_t)std::min<int64_t>(all - y0, Q4_GRID_Y));
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(MV_NT), 0, st, d, (const uint8_t*)rec, (const T*)x, xs, per, (int)y0, p.passes,
                               p.cb, p.chunks, p.range, out, stride);
        };
        if (p.mfma)
            hipLaunchKernelGGL(q4_mfma_kernel<T>, grid, dim3(MM_NT), lds, st, d, (const uint8_t*)rec, (const T*)x, xs, per,
                               (int)y0, p.passes, p.chunks, p.range, out, stride);
        else if (p.nx == 1) go(q4_matvec_kernel<T, 1>);
        else if (p.nx == 2) go(q4_matvec_kernel<T, 2>);
        else go(q4_matvec_kernel<T, 4>);
    }
    return HTM_OK;
}

// How a row's blocks are shared out: runs of at most 64 blocks, or the whole
// record (up to 512) where no two rows share a matrix and every record comes
// from memory once; shorter runs until the chip's 256 CUs have a workgroup each.
// Measured, us (runs x threads; 480 outputs a head, patterns of 768 columns x 32 cells):
//   4,096 rows of one matrix, 1 head: 1 x 256 109, 1 x 512 132, 2 x 256 124
//   1,024 rows, 7 heads: 2 x 512 220, 1 x 1,024 262, 7 x 256 294
//   256 rows of own matrices, 7 heads: 1 x 1,024 84, 2 x 512 87, 3 x 256 88
//   64 rows, 7 heads: 4 x 512 28, 2 x 512 47, 1 x 1,024 78
//   1 row, 7 heads: 105 x 256 7.6, 21 x 512 7.9, 105 x 1,024 10.6
// and of 2,048 x 12, in the same order: 58, 82, 79; 99, 128, 135; 37, 39, 40; 15, 22, 35;
// 8.1, 9.5, 11.5.
template <bool SOFTMAX>
static int q4_rows_launch(const Q4Dims& d, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows, int per,
                          const int32_t* live, float* out, hipStream_t st) {
    const int total = d.nh * d.nblk;
    int cblk;
    if (SOFTMAX) {
        // whole heads, as many as leave the chip's CUs a workgroup each (2,048 x 12 cells, 7 x 480, us: 36 rows 1 head 14.3,
        // 2 16.4, 4 25.1; 128 rows 28.2, 25.4, 25.9)
        const int64_t heads = ((int64_t)n_rows * d.nh + 255) / 256;
        cblk = d.nblk * (int)std::max<int64_t>(1, std::min<int64_t>(heads, std::min(d.nh, 64 / d.nblk)));
    } else {
        int chunks = per == 1 && total <= 512 ? 1 : (total + 63) / 64;
        chunks = std::min(total, std::max(chunks, 256 / n_rows));
        cblk = (total + chunks - 1) / chunks;
    }
    const int chunks = (total + cblk - 1) / cblk;
    const bool few = (int64_t)n_rows * chunks <= 256;
    const int nt = cblk > 64 ? 1024 : cblk > 24 || (few && cblk > 4) ? 512 : 256;
    const size_t lds = (16 * (size_t)(nt + 1) + (SOFTMAX ? (size_t)cblk * Q4_BLK : 0)) * sizeof(float);
    const auto kernel = q4_rows_kernel<SOFTMAX>;
    static std::atomic<uint64_t> raised{0};  // devices whose limit of dynamic LDS is raised
    if (int r = q4_raise_lds((const void*)kernel, lds, raised)) return r;
    for (int32_t r0 = 0; r0 < n_rows; r0 += Q4_GRID_Y)
        hipLaunchKernelGGL(kernel, dim3(chunks, n_rows - r0 < Q4_GRID_Y ? n_rows - r0 : Q4_GRID_Y), dim3(nt), lds, st, d,
                           (const uint8_t*)rec, pat, ps, per, r0, cblk, live, out);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 rows launch failed");
}

extern "C" {

int htm_q4_logits(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows, float* out,
                  void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_bitmap(s, rec, pat, ps, n_rows, out, __func__, &d, &per)) return r;
    if (!n_rows) return HTM_OK;
    return q4_rows_launch<false>(d, rec, pat, ps, n_rows, per, nullptr, out, (hipStream_t)stream);
}

int htm_q4_probabilities(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, const int32_t* live,
                         int32_t n_rows, float* out, void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_bitmap(s, rec, pat, ps, n_rows, out, __func__, &d, &per)) return r;
    if (d.no > Q4_MAX_SOFTMAX)
        return htm_fail(HTM_E_INVALID, "%s: at most %d outputs a head", __func__, Q4_MAX_SOFTMAX);
    if (!n_rows) return HTM_OK;
    hipStream_t st = (hipStream_t)stream;
    if (d.nblk <= 4 || (int64_t)n_rows * d.nh >= (d.nblk <= 16 ? 100 : 256))
        return q4_rows_launch<true>(d, rec, pat, ps, n_rows, per, live, out, st);
    // too few heads to fill the chip: the products in shorter runs, then the softmax.  One launch and two, us, Python call
    // included: 64 rows, 65,536 inputs, 1,000 outputs 30 and 19; 255 rows 32 and 34; 2,048 x 12 cells, 480 outputs, 16 rows
    // 13.0 and 12.2, 128 rows 13.1 and 14.2; 768 x 32 cells, 100 outputs, 4 rows 12.6 and 12.0
    if (int r = q4_rows_launch<false>(d, rec, pat, ps, n_rows, per, nullptr, out, st)) return r;
    const int64_t k = (int64_t)n_rows * d.nh;
    hipLaunchKernelGGL(q4_softmax_kernel, dim3((uint32_t)((k + Q4_NT / 64 - 1) / (Q4_NT / 64))), dim3(Q4_NT), 0, st, d, live,
                       per, k, out);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 softmax launch failed");
}

size_t htm_q4_work_bytes(const htm_q4_shape* s, int32_t n_rows) {
    Q4Dims d;
    int per;
    if (q4_dims(s, __func__, &d) || q4_rows(d, n_rows, __func__, &per) || !n_rows) return 0;
    const MvPlan p = mv_plan(d, per);
    return p.splits > 1 ? (size_t)p.splits * n_rows * d.nh * d.no * sizeof(float) : 0;
}

int htm_q4_matvec(const htm_q4_shape* s, const void* rec, const void* x, int32_t dtype, int64_t xs, int32_t n_rows,
                  float* out, void* work, size_t work_bytes, void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_dims(s, __func__, &d)) return r;
    if (int r = q4_rows(d, n_rows, __func__, &per)) return r;
    if (dtype != HTM_T_F32 && dtype != HTM_T_F16 && dtype != HTM_T_BF16)
        return htm_fail(HTM_E_INVALID, "%s: d_x must be float32, float16 or bfloat16", __func__);
    if (!n_rows) return HTM_OK;
    if (int r = q4_aligned(rec, __func__)) return r;
    if (!x || !out || (n_rows > 1 && xs < d.ni)) return htm_fail(HTM_E_INVALID, "%s: invalid argument", __func__);
    const MvPlan p = mv_plan(d, per);
    const int64_t n = (int64_t)n_rows * d.nh * d.no;
    if (p.splits > 1 && (!work || (uintptr_t)work % 4 || work_bytes < (size_t)(p.splits * n) * sizeof(float)))
        return htm_fail(HTM_E_INVALID, "%s: needs htm_q4_work_bytes of scratch", __func__);
    hipStream_t st = (hipStream_t)stream;
    float* y = p.splits > 1 ? (float*)work : out;
    const int r = dtype == HTM_T_F32   ? mv_launch<float>(p, d, rec, x, xs, per, y, n, st)
                  : dtype == HTM_T_F16 ? mv_launch<__half>(p, d, rec, x, xs, per, y, n, st)
                                       : mv_launch<__hip_bfloat16>(p, d, rec, x, xs, per, y, n, st);
    if (r) return r;
    if (p.splits > 1)
        hipLaunchKernelGGL(q4_join_kernel, dim3((uint32_t)((n + 63) / 64)), dim3(256), 0, st, y, p.splits, n, out);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 matvec launch failed");
}

}  // extern "C"
