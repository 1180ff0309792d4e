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

#include "htm_dev.h"
#include "q4_dev.h"

#define Q4_NT 256

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
// One thread per group of one (model, input, head): two passes over its
// weights, the largest magnitude and then the codes.
template <typename T>
__global__ void __launch_bounds__(Q4_NT) q4_quantise_kernel(Q4Dims d, const T* __restrict__ w, int64_t ms, int64_t is,
                                                            int64_t hs, uint8_t* __restrict__ rec, int32_t* bad) {
    const int64_t per = (int64_t)d.nh * d.ngrp;
    const int64_t total = (int64_t)d.nm * d.ni * per;
    for (int64_t t = (int64_t)blockIdx.x * Q4_NT + threadIdx.x; t < total; t += (int64_t)gridDim.x * Q4_NT) {
        const int64_t row = t / per;
        const int k = (int)(t - row * per), h = k / d.ngrp, g = k - h * d.ngrp;
        const T* src = w + (row / d.ni) * ms + (row % d.ni) * is + (int64_t)h * hs;
        const int o0 = g * d.group, o1 = min(o0 + d.group, d.nblk * Q4_BLK);
        double amax = 0.0;
        bool odd = false;
        for (int o = o0; o < min(o1, d.no); o++) {
            const double a = fabs((double)src[o]);
            odd |= !(a <= 1.7976931348623157e308);
            amax = fmax(amax, a);
        }
        // (past the bfloat16 range on either side: no scale for the group's largest weight)
        odd |= amax > 2.3e39;
        const float s0 = (float)(amax / 7.0);
        const uint32_t sb = s0 >= 1.17549435e-38f && !odd ? bf16_round(s0) : 0u;
        const double s = (double)bf16_up(sb);
        uint8_t* r = rec + row * (int64_t)d.pitch;
        for (int o = o0; o < o1; o += 2) {
            uint32_t c[2] = {8u, 8u};
            for (int j = 0; j < 2; j++)
                if (o + j < d.no && s > 0.0) {
                    const double q = fmin(fmax(rint((double)src[o + j] / s), -7.0), 7.0);
                    c[j] = (uint32_t)(8 + (int)q);
                }
            r[((size_t)h * d.nblk * Q4_BLK + o) >> 1] = (uint8_t)(c[0] | (c[1] << 4));
        }
        reinterpret_cast<uint16_t*>(r + d.scales)[h * d.ngrp + g] = (uint16_t)sb;
        if (odd) *bad = 1;
    }
}

int q4_quantise_launch(const Q4Dims& d, const void* w, int32_t dtype, int64_t ms, int64_t is, int64_t hs, void* rec,
                       int32_t* bad, hipStream_t st) {
    const int64_t total = (int64_t)d.nm * d.ni * d.nh * d.ngrp;
    const int64_t wg = (total + Q4_NT - 1) / Q4_NT;
    const dim3 grid((uint32_t)(wg < 65536 ? wg : 65536));
    if (dtype == HTM_T_F64)
        hipLaunchKernelGGL(q4_quantise_kernel<double>, grid, dim3(Q4_NT), 0, st, d, (const double*)w, ms, is, hs,
                           (uint8_t*)rec, bad);
    else
        hipLaunchKernelGGL(q4_quantise_kernel<float>, grid, dim3(Q4_NT), 0, st, d, (const float*)w, ms, is, hs,
                           (uint8_t*)rec, bad);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 quantise launch failed");
}

// ------------------------------------------------------------------ products
// A record's block: 32 outputs' codes in 16 bytes, under one scale.  A code's
// four bits lie in the low mantissa bits of a 16-bit float of exponent zero:
// masked there they are the number code * 2^-24 (bits 0-3) or code * 2^-20
// (bits 4-7), a subnormal float16 that a mixed-precision FMA reads exactly --
// one mask and one FMA a weight, 13 instructions per 8 weights with the shift
// (shift, convert and FMA apart: 24).  The sum of scale * code is corrected by
// 8 * sum of scales once at the end.
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ half2_t as_half2(uint32_t u) { return __builtin_bit_cast(half2_t, u); }

struct Q4Acc {
    float v[Q4_BLK];
    float s;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < Q4_BLK; j++) v[j] = 0.0f;
        s = 0.0f;
    }
    // + m * (codes), m the scale times the input's number
    __device__ __forceinline__ void add(uint4 c, float m) {
        const float m0 = m * 16777216.0f, m1 = m * 1048576.0f;
        s += m;
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t u = w[k], h = w[k] >> 8;
            const half2_t a = as_half2(u & 0x000F000Fu), b = as_half2(u & 0x00F000F0u);
            const half2_t d = as_half2(h & 0x000F000Fu), e = as_half2(h & 0x00F000F0u);
            float* p = v + k * 8;
            p[0] = __builtin_fmaf((float)a.x, m0, p[0]);
            p[1] = __builtin_fmaf((float)b.x, m1, p[1]);
            p[2] = __builtin_fmaf((float)d.x, m0, p[2]);
            p[3] = __builtin_fmaf((float)e.x, m1, p[3]);
            p[4] = __builtin_fmaf((float)a.y, m0, p[4]);
            p[5] = __builtin_fmaf((float)b.y, m1, p[5]);
            p[6] = __builtin_fmaf((float)d.y, m0, p[6]);
            p[7] = __builtin_fmaf((float)e.y, m1, p[7]);
        }
    }
};

// The workgroup's threads are slots x blocks: thread (slot, block) has summed
// its share of the inputs for one block's 32 outputs.  Sums over the slots, in
// a fixed order, through LDS (16 of the 32 at a time); put(output, y) is called
// once for each of the workgroup's nblk * 32 outputs.
template <int NT, typename PUT>
__device__ __forceinline__ void q4_join(Q4Acc& a, int nblk, int slots, float (*sm)[NT + 1], PUT put) {
    const int nout = nblk * 16;
    const int parts = nout < NT ? NT / nout : 1;
    const float off = 8.0f * a.s;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 16; j++) sm[j][threadIdx.x] = a.v[half * 16 + j] - off;
        __syncthreads();
        if (parts == 1) {
            for (int o = threadIdx.x; o < nout; o += NT) {
                float y = 0.0f;
                for (int s = 0; s < slots; s++) y += sm[o & 15][s * nblk + (o >> 4)];
                put((o >> 4) * Q4_BLK + half * 16 + (o & 15), y);
            }
        } else {  // few outputs: several threads each take a run of slots, then one adds up theirs
            const int part = threadIdx.x / nout, o = threadIdx.x - part * nout;
            const int each = (slots + parts - 1) / parts;
            float y = 0.0f;
            if (part < parts)
                for (int s = part * each; s < min(slots, part * each + each); s++) y += sm[o & 15][s * nblk + (o >> 4)];
            __syncthreads();
            float* flat = &sm[0][0];
            if (part < parts) flat[threadIdx.x] = y;
            __syncthreads();
            if (threadIdx.x < (uint32_t)nout) {
                y = 0.0f;
                for (int p = 0; p < parts; p++) y += flat[p * nout + o];
                put((o >> 4) * Q4_BLK + half * 16 + (o & 15), y);
            }
        }
    }
}

#define Q4_LIST 2048  // active inputs listed at a time

// Word bitmaps.  One workgroup per (row, head, chunk of the head's blocks): the
// active inputs are listed in LDS in ascending order, and each slot of threads
// reads the records of every slots-th run of four, all blocks of the chunk side
// by side.  SOFTMAX: the chunk is the whole head, whose probabilities are
// written instead.
template <int NT, bool SOFTMAX>
__global__ void __launch_bounds__(NT) q4_rows_kernel(Q4Dims d, const uint8_t* __restrict__ rec,
                                                     const uint32_t* __restrict__ pat, int64_t ps, int per_model,
                                                     int row0, int chunks, int cblk, const int32_t* __restrict__ live,
                                                     float* __restrict__ out) {
    __shared__ float sm[16][NT + 1];
    __shared__ __attribute__((aligned(8))) uint16_t list[Q4_LIST];
    __shared__ uint32_t wsum[NT / 64];
    __shared__ float y_sh[SOFTMAX ? Q4_MAX_SOFTMAX : 1];
    const int row = row0 + blockIdx.y;
    const int h = blockIdx.x / chunks, b0 = (blockIdx.x - h * chunks) * cblk;
    const int nblk = min(cblk, d.nblk - b0);
    const int slots = NT / nblk;
    const int slot = threadIdx.x / nblk, b = threadIdx.x - slot * nblk;
    const uint32_t* p = pat + (int64_t)row * ps;
    const int words = d.ni / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    // the thread's words, their set bits' place among all
    const int each = (words + NT - 1) / NT;
    const int w0 = min(words, (int)threadIdx.x * each), w1 = min(words, w0 + each);
    uint32_t mine = 0;
    for (int w = w0; w < w1; w++) mine += __popc(p[w]);
    uint32_t at = mine;
    for (int k = 1; k < 64; k <<= 1) {
        const uint32_t o = __shfl_up(at, k);
        if (lane >= k) at += o;
    }
    if (lane == 63) wsum[wave] = at;
    __syncthreads();
    uint32_t n = 0;
    at -= mine;
    for (int k = 0; k < NT / 64; k++) {
        if (k < wave) at += wsum[k];
        n += wsum[k];
    }

    Q4Acc acc;
    acc.clear();
    const int blk = h * d.nblk + b0 + b;
    const uint8_t* base = rec + (int64_t)(row / per_model) * d.ni * d.pitch;
    const uint32_t c_off = (uint32_t)blk * 16u;
    const uint32_t s_off = d.scales + 2u * (uint32_t)(h * d.ngrp + (b0 + b) * Q4_BLK / d.group);
    for (uint32_t r0 = 0; r0 < n; r0 += Q4_LIST) {  // (a second round only beyond Q4_LIST active inputs)
        if (r0) __syncthreads();
        uint32_t k = at;
        for (int w = w0; w < w1; w++) {
            uint32_t x = p[w];
            while (x) {
                const uint32_t q = k++ - r0;
                if (q < Q4_LIST) list[q] = (uint16_t)(w * 32 + __ffs(x) - 1);
                x &= x - 1;
            }
        }
        __syncthreads();
        const int m = (int)min(n - r0, (uint32_t)Q4_LIST);
        if (slot < slots)
            for (int i = slot * 4; i < m; i += slots * 4) {
                const uint2 e = *reinterpret_cast<const uint2*>(list + i);
                const uint32_t idx[4] = {e.x & 0xFFFFu, e.x >> 16, e.y & 0xFFFFu, e.y >> 16};
                uint4 c[4];
                float s[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    // (behind the list's end: the run's first record again, times zero)
                    const uint8_t* r = base + (uint64_t)(i + u < m ? idx[u] : idx[0]) * d.pitch;
                    c[u] = *reinterpret_cast<const uint4*>(r + c_off);
                    const float v = bf16_up(*reinterpret_cast<const uint16_t*>(r + s_off));
                    s[u] = i + u < m ? v : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < 4; u++) acc.add(c[u], s[u]);
            }
    }
    float* o = out + ((int64_t)row * d.nh + h) * d.no;
    const int first = b0 * Q4_BLK;
    if (!SOFTMAX) {
        q4_join<NT>(acc, nblk, slots, sm, [&](int k, float y) {
            if (first + k < d.no) o[first + k] = y;
        });
        return;
    }
    q4_join<NT>(acc, nblk, slots, sm, [&](int k, float y) { y_sh[k] = y; });
    __syncthreads();
    int nl = d.no;
    if (live) nl = min(max(live[row / per_model], 0), d.no);
    float* red = &sm[0][0];
    float m = -INFINITY;
    for (int k = threadIdx.x; k < nl; k += NT) m = fmaxf(m, y_sh[k]);
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    if (lane == 0) red[wave] = m;
    __syncthreads();
    for (int k = 0; k < NT / 64; k++) m = fmaxf(m, red[k]);
    constexpr int PER = (Q4_MAX_SOFTMAX + NT - 1) / NT;
    float e[PER], t = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int k = threadIdx.x + j * NT;
        e[j] = k < nl ? expf(y_sh[k] - m) : 0.0f;
        t += e[j];
    }
    for (int k = 32; k; k >>= 1) t += __shfl_xor(t, k);
    if (lane == 0) red[64 + wave] = t;
    __syncthreads();
    t = 0.0f;
    for (int k = 0; k < NT / 64; k++) t += red[64 + k];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int k = threadIdx.x + j * NT;
        if (k < d.no) o[k] = k < nl ? e[j] / t : 0.0f;
    }
}

// One thread per output: every input in turn.
__device__ __forceinline__ float q4_weight(const uint8_t* __restrict__ r, const Q4Dims& d, int h, int o) {
    const int at = h * d.nblk * Q4_BLK + o;
    const int c = (r[at >> 1] >> ((at & 1) * 4)) & 15;
    const uint32_t s = reinterpret_cast<const uint16_t*>(r + d.scales)[h * d.ngrp + o / d.group];
    return bf16_up(s) * (float)(c - 8);
}

template <typename T>
__global__ void __launch_bounds__(Q4_NT) q4_matvec_kernel(Q4Dims d, const uint8_t* __restrict__ rec,
                                                          const T* __restrict__ x, int64_t xs, int per_model,
                                                          int row0, float* __restrict__ out) {
    const int row = row0 + blockIdx.y;
    const int k = blockIdx.x * Q4_NT + threadIdx.x;
    if (k >= d.nh * d.no) return;
    const int h = k / d.no, o = k - h * d.no;
    const uint8_t* base = rec + (int64_t)(row / per_model) * d.ni * d.pitch;
    const T* v = x + (int64_t)row * xs;
    float acc = 0.0f;
    for (int i = 0; i < d.ni; i++) acc = fmaf(x_up(v[i]), q4_weight(base + (int64_t)i * d.pitch, d, h, o), acc);
    out[(int64_t)row * d.nh * d.no + k] = acc;
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

// Chunks of a head and the workgroup's width.  Many rows: whole heads (up to 32
// blocks) by 256 threads.  Few workgroups: 1,024 threads each, and logits in
// chunks down to one block until the chip's 256 CUs have one each, since then a
// row's time is its longest chain of record reads.
template <bool SOFTMAX>
static void q4_rows_launch(const Q4Dims& d, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows, int per,
                           const int32_t* live, float* out, hipStream_t st) {
    int chunks = (d.nblk + 31) / 32;
    const bool wide = (int64_t)n_rows * d.nh * chunks < 512;
    if (wide && !SOFTMAX)
        while (chunks < d.nblk && (int64_t)n_rows * d.nh * chunks < 256) chunks++;
    const int cblk = (d.nblk + chunks - 1) / chunks;
    chunks = (d.nblk + cblk - 1) / cblk;
    for (int32_t r0 = 0; r0 < n_rows; r0 += Q4_GRID_Y) {
        const dim3 grid(d.nh * chunks, n_rows - r0 < Q4_GRID_Y ? n_rows - r0 : Q4_GRID_Y);
        if (wide)
            hipLaunchKernelGGL((q4_rows_kernel<1024, SOFTMAX>), grid, dim3(1024), 0, st, d, (const uint8_t*)rec, pat, ps,
                               per, r0, chunks, cblk, live, out);
        else
            hipLaunchKernelGGL((q4_rows_kernel<256, SOFTMAX>), grid, dim3(256), 0, st, d, (const uint8_t*)rec, pat, ps,
                               per, r0, chunks, cblk, live, out);
    }
}

extern "C" {

int htm_q4_logits(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows, float* out,
                  void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_bitmap(s, rec, pat, ps, n_rows, out, __func__, &d, &per)) return r;
    if (!n_rows) return HTM_OK;
    q4_rows_launch<false>(d, rec, pat, ps, n_rows, per, nullptr, out, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 logits launch failed");
}

int htm_q4_probabilities(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, const int32_t* live,
                         int32_t n_rows, float* out, void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_bitmap(s, rec, pat, ps, n_rows, out, __func__, &d, &per)) return r;
    if (d.no > Q4_MAX_SOFTMAX)
        return htm_fail(HTM_E_INVALID, "%s: at most %d outputs a head", __func__, Q4_MAX_SOFTMAX);
    if (!n_rows) return HTM_OK;
    q4_rows_launch<true>(d, rec, pat, ps, n_rows, per, live, out, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 probabilities launch failed");
}

size_t htm_q4_work_bytes(const htm_q4_shape* s, int32_t n_rows) {
    Q4Dims d;
    (void)n_rows;
    return q4_dims(s, __func__, &d) ? 0 : 0;
}

int htm_q4_matvec(const htm_q4_shape* s, const void* rec, const void* x, int32_t dtype, int64_t xs, int32_t n_rows,
                  float* out, void* work, size_t work_bytes, void* stream) {
    Q4Dims d;
    int per;
    (void)work;
    (void)work_bytes;
    if (int r = q4_dims(s, __func__, &d)) return r;
    if (int r = q4_rows(d, n_rows, __func__, &per)) return r;
    if (dtype != HTM_T_F32 && dtype != HTM_T_F16 && dtype != HTM_T_BF16)
        return htm_fail(HTM_E_INVALID, "%s: d_x must be float32, float16 or bfloat16", __func__);
    if (!n_rows) return HTM_OK;
    if (int r = q4_aligned(rec, __func__)) return r;
    if (!x || !out || (n_rows > 1 && xs < d.ni)) return htm_fail(HTM_E_INVALID, "%s: invalid argument", __func__);
    hipStream_t st = (hipStream_t)stream;
    for (int32_t r0 = 0; r0 < n_rows; r0 += Q4_GRID_Y) {
        const dim3 grid((d.nh * d.no + Q4_NT - 1) / Q4_NT, n_rows - r0 < Q4_GRID_Y ? n_rows - r0 : Q4_GRID_Y);
        if (dtype == HTM_T_F32)
            hipLaunchKernelGGL(q4_matvec_kernel<float>, grid, dim3(Q4_NT), 0, st, d, (const uint8_t*)rec,
                               (const float*)x, xs, per, r0, out);
        else if (dtype == HTM_T_F16)
            hipLaunchKernelGGL(q4_matvec_kernel<__half>, grid, dim3(Q4_NT), 0, st, d, (const uint8_t*)rec,
                               (const __half*)x, xs, per, r0, out);
        else
            hipLaunchKernelGGL(q4_matvec_kernel<__hip_bfloat16>, grid, dim3(Q4_NT), 0, st, d, (const uint8_t*)rec,
                               (const __hip_bfloat16*)x, xs, per, r0, out);
    }
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 matvec launch failed");
}

}  // extern "C"
