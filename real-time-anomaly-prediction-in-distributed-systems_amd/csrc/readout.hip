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
// One thread per output: every input in turn.
__device__ __forceinline__ float q4_weight(const uint8_t* __restrict__ r, const Q4Dims& d, int h, int o) {
    const int at = h * d.nblk * Q4_BLK + o;
    const int c = (r[at >> 1] >> ((at & 1) * 4)) & 15;
    const uint32_t s = reinterpret_cast<const uint16_t*>(r + d.scales)[h * d.ngrp + o / d.group];
    return bf16_up(s) * (float)(c - 8);
}

__global__ void __launch_bounds__(Q4_NT) q4_logits_kernel(Q4Dims d, const uint8_t* __restrict__ rec,
                                                          const uint32_t* __restrict__ pat, int64_t ps, int per_model,
                                                          int row0, float* __restrict__ out) {
    const int row = row0 + blockIdx.y;
    const int k = blockIdx.x * Q4_NT + threadIdx.x;
    if (k >= d.nh * d.no) return;
    const int h = k / d.no, o = k - h * d.no;
    const uint8_t* base = rec + (int64_t)(row / per_model) * d.ni * d.pitch;
    const uint32_t* p = pat + (int64_t)row * ps;
    float acc = 0.0f;
    for (int w = 0; w < d.ni / 32; w++) {
        uint32_t x = p[w];
        while (x) {
            const int i = w * 32 + __ffs(x) - 1;
            x &= x - 1;
            acc += q4_weight(base + (int64_t)i * d.pitch, d, h, o);
        }
    }
    out[(int64_t)row * d.nh * d.no + k] = acc;
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

// softmax over each (row, head)'s live outputs, in place: one workgroup each
__global__ void __launch_bounds__(Q4_NT) q4_softmax_kernel(Q4Dims d, const int32_t* __restrict__ live, int per_model,
                                                           int row0, float* __restrict__ y) {
    __shared__ float red[Q4_NT / 64];
    const int row = row0 + blockIdx.y;
    float* p = y + ((int64_t)row * d.nh + blockIdx.x) * d.no;
    int n = d.no;
    if (live) n = min(max(live[row / per_model], 0), d.no);
    float m = -INFINITY;
    for (int o = threadIdx.x; o < n; o += Q4_NT) m = fmaxf(m, p[o]);
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int k = 0; k < Q4_NT / 64; k++) m = fmaxf(m, red[k]);
    __syncthreads();
    float e[Q4_MAX_SOFTMAX / Q4_NT], s = 0.0f;
#pragma unroll
    for (int j = 0; j < Q4_MAX_SOFTMAX / Q4_NT; j++) {
        const int o = threadIdx.x + j * Q4_NT;
        e[j] = o < n ? expf(p[o] - m) : 0.0f;
        s += e[j];
    }
    for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0f;
    for (int k = 0; k < Q4_NT / 64; k++) s += red[k];
#pragma unroll
    for (int j = 0; j < Q4_MAX_SOFTMAX / Q4_NT; j++) {
        const int o = threadIdx.x + j * Q4_NT;
        if (o < d.no) p[o] = o < n ? e[j] / s : 0.0f;
    }
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

#define Q4_GRID_Y 65535  // rows of one launch

static int q4_logits_launch(const Q4Dims& d, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows, int per,
                            float* out, hipStream_t st) {
    for (int32_t r0 = 0; r0 < n_rows; r0 += Q4_GRID_Y) {
        const dim3 grid((d.nh * d.no + Q4_NT - 1) / Q4_NT, n_rows - r0 < Q4_GRID_Y ? n_rows - r0 : Q4_GRID_Y);
        hipLaunchKernelGGL(q4_logits_kernel, grid, dim3(Q4_NT), 0, st, d, (const uint8_t*)rec, pat, ps, per, r0, out);
    }
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 logits launch failed");
}

int htm_q4_logits(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, int32_t n_rows, float* out,
                  void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_bitmap(s, rec, pat, ps, n_rows, out, __func__, &d, &per)) return r;
    return n_rows ? q4_logits_launch(d, rec, pat, ps, n_rows, per, out, (hipStream_t)stream) : HTM_OK;
}

int htm_q4_probabilities(const htm_q4_shape* s, const void* rec, const uint32_t* pat, int64_t ps, const int32_t* live,
                         int32_t n_rows, float* out, void* stream) {
    Q4Dims d;
    int per;
    if (int r = q4_bitmap(s, rec, pat, ps, n_rows, out, __func__, &d, &per)) return r;
    if (d.no > Q4_MAX_SOFTMAX)
        return htm_fail(HTM_E_INVALID, "%s: at most %d outputs a head", __func__, Q4_MAX_SOFTMAX);
    if (!n_rows) return HTM_OK;
    if (int r = q4_logits_launch(d, rec, pat, ps, n_rows, per, out, (hipStream_t)stream)) return r;
    for (int32_t r0 = 0; r0 < n_rows; r0 += Q4_GRID_Y) {
        const dim3 grid(d.nh, n_rows - r0 < Q4_GRID_Y ? n_rows - r0 : Q4_GRID_Y);
        hipLaunchKernelGGL(q4_softmax_kernel, grid, dim3(Q4_NT), 0, (hipStream_t)stream, d, live, per, r0, out);
    }
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "q4 softmax launch failed");
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
