// beam.hip -- beam selection over beams x buckets, and the beams' states
// reordered by parent.  The reference's look-ahead feeds one value seven times
// (ML/HTM/ModelTesting.py:66-72); a forecast that follows its own predictions
// keeps several continuations of every stream and drops the worse ones.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "beam_dev.h"
#include "htm_dev.h"

#define BS_NT 256
#define BS_MAX 64  // beams

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(__hip_bfloat16 v) { return __bfloat162float(v); }

// (score, place) as one unsigned key: larger is better, equal scores by the
// lower place; 0: never taken
__device__ __forceinline__ uint64_t cand_key(float s, uint32_t place) {
    s += 0.0f;  // -0 and 0 are the same score
    if (!(s > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(s);
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((uint64_t)o << 32) | (0xFFFFFFFFu - place);
}

__device__ __forceinline__ float key_score(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

struct SelArgs {
    const void* x;
    int64_t gs, bs;
    const float* score;
    const int32_t* live;
    int32_t win, wout, v;
    float* o_score;
    int32_t* o_parent;
    int32_t* o_bucket;
};

// One workgroup per group: every beam's log-sum-exp, then the best key below
// the last one taken, n_beams times.
template <typename T>
__global__ void __launch_bounds__(BS_NT) beam_select_kernel(SelArgs a) {
    __shared__ double base[BS_MAX];  // score - log(sum)
    __shared__ float top[BS_MAX];
    __shared__ uint64_t red[BS_NT / 64];
    const int g = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const T* x = (const T*)a.x + (int64_t)g * a.gs;
    int n = a.v;
    if (a.live) n = min(max(a.live[g], 0), a.v);
    for (int w = wave; w < a.win; w += BS_NT / 64) {
        const T* p = x + (int64_t)w * a.bs;
        float m = -INFINITY;
        for (int o = lane; o < n; o += 64) m = fmaxf(m, up(p[o]));
        for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
        double s = 0.0;
        for (int o = lane; o < n; o += 64) s += exp((double)up(p[o]) - (double)m);
        for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
        // (no finite logit, an infinite one or a NaN: the sum is 0 or NaN, and no score of the beam is a number)
        if (lane == 0) {
            base[w] = (double)a.score[(int64_t)g * a.win + w] - log(s);
            top[w] = m;
        }
    }
    __syncthreads();
    uint64_t prev = ~0ull;
    for (int j = 0; j < a.wout; j++) {
        uint64_t best = 0;
        for (int w = 0; w < a.win; w++)
            for (int o = threadIdx.x; o < n; o += BS_NT) {
                const float s = (float)(((double)up(x[(int64_t)w * a.bs + o]) - (double)top[w]) + base[w]);
                const uint64_t k = cand_key(s, (uint32_t)(w * a.v + o));
                if (k < prev && k > best) best = k;
            }
        for (int k = 32; k; k >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, k);
            best = other > best ? other : best;
        }
        if (lane == 0) red[wave] = best;
        __syncthreads();
        for (int k = 0; k < BS_NT / 64; k++) best = red[k] > best ? red[k] : best;
        __syncthreads();
        if (threadIdx.x == 0) {
            const int64_t at = (int64_t)g * a.wout + j;
            const uint32_t place = 0xFFFFFFFFu - (uint32_t)best;
            a.o_score[at] = best ? key_score(best) : -INFINITY;
            a.o_parent[at] = best ? (int32_t)(place / (uint32_t)a.v) : min(j, a.win - 1);
            a.o_bucket[at] = best ? (int32_t)(place % (uint32_t)a.v) : -1;
        }
        prev = best;
    }
}

// ------------------------------------------------------------------- rows
// Out of place: a grid-stride copy in units of U, the row of each unit found
// by division.
template <typename U>
__global__ void __launch_bounds__(256) rows_copy_kernel(const U* __restrict__ src, U* __restrict__ dst, uint64_t per,
                                                        const int32_t* __restrict__ idx, int64_t n_rows, int beams,
                                                        int64_t n_src) {
    const uint64_t total = per * (uint64_t)n_rows;
    for (uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (uint64_t)gridDim.x * 256) {
        const uint64_t r = t / per, k = t - r * per;
        int64_t from = idx[r];
        if (beams) {
            const int64_t w = (int64_t)(r % (uint64_t)beams);
            from = (int64_t)r - w + (from >= 0 && from < beams ? from : w);
        } else if (from < 0 || from >= n_src) {
            continue;
        }
        dst[t] = src[(uint64_t)from * per + k];
    }
}

// In place: a thread owns one unit column of a group, reads it for every beam
// and only then writes it, so no other thread's data is involved.
template <typename U>
__global__ void __launch_bounds__(256) rows_inplace_kernel(U* base, uint64_t per, const int32_t* __restrict__ idx,
                                                           int64_t groups, int beams) {
    const uint64_t total = per * (uint64_t)groups;
    for (uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (uint64_t)gridDim.x * 256) {
        const uint64_t g = t / per, k = t - g * per;
        const int32_t* p = idx + g * (uint64_t)beams;
        U* b = base + g * (uint64_t)beams * per + k;
        U v[BS_MAX];
#pragma unroll
        for (int w = 0; w < BS_MAX; w++)
            if (w < beams) {
                const int q = p[w];
                if (q >= 0 && q < beams && q != w) v[w] = b[(uint64_t)q * per];
            }
#pragma unroll
        for (int w = 0; w < BS_MAX; w++)
            if (w < beams) {
                const int q = p[w];
                if (q >= 0 && q < beams && q != w) b[(uint64_t)w * per] = v[w];
            }
    }
}

template <typename U>
static void rows_launch(const RowMoves& m, int k, const int32_t* idx, int64_t n_rows, int32_t beams, int64_t n_src,
                        hipStream_t st) {
    const uint64_t per = m.bytes[k] / sizeof(U);
    const bool inplace = m.src[k] == m.dst[k];
    const uint64_t total = per * (uint64_t)(inplace ? n_rows / beams : n_rows);
    const uint64_t wg = (total + 255) / 256;
    const dim3 grid((uint32_t)(wg < 65536 ? wg : 65536));
    if (inplace)
        hipLaunchKernelGGL(rows_inplace_kernel<U>, grid, dim3(256), 0, st, (U*)m.dst[k], per, idx, n_rows / beams, beams);
    else
        hipLaunchKernelGGL(rows_copy_kernel<U>, grid, dim3(256), 0, st, (const U*)m.src[k], (U*)m.dst[k], per, idx,
                           n_rows, beams, n_src);
}

int rows_move(const RowMoves& m, const int32_t* idx, int64_t n_rows, int32_t beams, int64_t n_src, hipStream_t st) {
    if (!n_rows) return HTM_OK;
    for (int k = 0; k < m.n; k++) {
        if (!m.bytes[k]) continue;
        const uint64_t a = m.bytes[k] | (uint64_t)(uintptr_t)m.src[k] | (uint64_t)(uintptr_t)m.dst[k];
        if (a % 4 == 0) rows_launch<uint32_t>(m, k, idx, n_rows, beams, n_src, st);
        else rows_launch<uint8_t>(m, k, idx, n_rows, beams, n_src, st);
    }
    return hipGetLastError() == hipSuccess ? HTM_OK : htm_fail(HTM_E_HIP, "row move launch failed");
}

extern "C" {

size_t htm_beam_work_bytes(int32_t n_groups, int32_t beams_in, int32_t n_beams, int32_t n_outputs) {
    (void)n_groups; (void)beams_in; (void)n_beams; (void)n_outputs;
    return 0;
}

int htm_beam_select(const void* x, int32_t dtype, int64_t gs, int64_t bs, const float* score, const int32_t* live,
                    int32_t groups, int32_t win, int32_t wout, int32_t v, float* o_score, int32_t* o_parent,
                    int32_t* o_bucket, void* work, size_t work_bytes, void* stream) {
    (void)work;
    (void)work_bytes;
    if (groups < 0 || win < 1 || win > BS_MAX || wout < 1 || wout > BS_MAX || v < 1 || (int64_t)win * v >= 0x7FFFFFFFll)
        return htm_fail(HTM_E_INVALID, "%s: 1..64 beams in and out, outputs >= 1, beams_in * outputs < 2^31", __func__);
    if (dtype != HTM_T_F32 && dtype != HTM_T_F16 && dtype != HTM_T_BF16)
        return htm_fail(HTM_E_INVALID, "%s: d_logits must be float32, float16 or bfloat16", __func__);
    if (!groups) return HTM_OK;
    if (!x || !score || !o_score || !o_parent || !o_bucket || gs < 0 || bs < 0)
        return htm_fail(HTM_E_INVALID, "%s: invalid argument", __func__);
    const SelArgs a{x, gs, bs, score, live, win, wout, v, o_score, o_parent, o_bucket};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == HTM_T_F32)
        hipLaunchKernelGGL(beam_select_kernel<float>, dim3(groups), dim3(BS_NT), 0, st, a);
    else if (dtype == HTM_T_F16)
        hipLaunchKernelGGL(beam_select_kernel<__half>, dim3(groups), dim3(BS_NT), 0, st, a);
    else
        hipLaunchKernelGGL(beam_select_kernel<__hip_bfloat16>, dim3(groups), dim3(BS_NT), 0, st, a);
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
