// The head with the requests' low-rank adapters beside it (mk_head_logits in include/mako_b200.h), as two launches: the rows'
// down projections, then tiles of the logits with the up projections added before they are written.
#include "round_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mk {
namespace {

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// inner[row][r] = scale * down[a][r] . hidden[row], a warp each.
template <typename T>
__global__ void __launch_bounds__(256) head_inner_kernel(const mk_head h, const T* hidden, uint64_t hidden_ld,
                                                         const int32_t* adapter, float* inner)
{
    const uint32_t row = blockIdx.x, r = blockIdx.y * 8u + threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const int32_t a = adapter[row];
    if (a < 0 || (uint32_t)a >= h.n_adapters || r >= h.rank)
        return;
    const T* x = hidden + row * hidden_ld;
    const T* w = static_cast<const T*>(h.down) + ((size_t)a * h.rank + r) * h.dim;
    float sum = 0.0f;
    for (uint32_t i = lane; i < h.dim; i += 32)
        sum = fmaf(to_float(x[i]), to_float(w[i]), sum);
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
        sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0)
        inner[(size_t)row * kHeadMaxRank + r] = (h.scale ? h.scale[a] : 1.0f) * sum;
}

// 64 columns of 16 rows a CTA; a thread has four columns of one row.
template <typename T>
__global__ void __launch_bounds__(256) head_tile_kernel(const mk_head h, const T* hidden, uint64_t hidden_ld,
                                                        const int32_t* adapter, uint32_t rows, const float* inner, float* logits,
                                                        uint64_t ld)
{
    __shared__ float s_x[16][33], s_w[64][33];
    const uint32_t v0 = blockIdx.x * 64u, t0 = blockIdx.y * 16u, tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    const T* weight = static_cast<const T*>(h.weight);
    float acc[4] = {};
    for (uint32_t k0 = 0; k0 < h.dim; k0 += 32) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 16 * 32; i += 256) {
            const uint32_t t = t0 + i / 32, k = k0 + i % 32;
            s_x[i / 32][i % 32] = t < rows && k < h.dim ? to_float(hidden[t * hidden_ld + k]) : 0.0f;
        }
        for (uint32_t i = threadIdx.x; i < 64 * 32; i += 256) {
            const uint32_t v = v0 + i / 32, k = k0 + i % 32;
            s_w[i / 32][i % 32] = v < h.n_vocab && k < h.dim ? to_float(weight[(size_t)v * h.dim + k]) : 0.0f;
        }
        __syncthreads();
        for (uint32_t k = 0; k < 32; ++k)
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c)
                acc[c] = fmaf(s_x[ty][k], s_w[tx + 16 * c][k], acc[c]);
    }
    const uint32_t t = t0 + ty;
    if (t >= rows)
        return;
    const int32_t a = h.n_adapters ? adapter[t] : -1;
    for (uint32_t c = 0; c < 4; ++c) {
        const uint32_t v = v0 + tx + 16 * c;
        if (v >= h.n_vocab)
            continue;
        if (a >= 0 && (uint32_t)a < h.n_adapters) {
            const T* up = static_cast<const T*>(h.up) + ((size_t)a * h.n_vocab + v) * h.rank;
            float d = 0.0f;
            for (uint32_t r = 0; r < h.rank; ++r)
                d = fmaf(inner[(size_t)t * kHeadMaxRank + r], to_float(up[r]), d);
            acc[c] += d;
        }
        logits[t * ld + v] = acc[c];
    }
}

template <typename T>
cudaError_t launch(const mk_head& h, const void* hidden, uint64_t hidden_ld, const int32_t* adapter, uint32_t rows, float* inner,
                   float* logits, uint64_t ld, cudaStream_t stream)
{
    const T* x = static_cast<const T*>(hidden);
    if (h.n_adapters)
        head_inner_kernel<T><<<dim3(rows, (h.rank + 7) / 8), 256, 0, stream>>>(h, x, hidden_ld, adapter, inner);
    head_tile_kernel<T><<<dim3((h.n_vocab + 63) / 64, (rows + 15) / 16), 256, 0, stream>>>(h, x, hidden_ld, adapter, rows, inner,
                                                                                         logits, ld);
    return cudaGetLastError();
}

} // namespace

cudaError_t launch_head_logits(const mk_head& h, const void* hidden, uint64_t hidden_ld, const int32_t* adapter, uint32_t rows,
                               float* inner, float* logits, uint64_t ld, cudaStream_t stream)
{
    return h.type == MK_BF16 ? launch<__nv_bfloat16>(h, hidden, hidden_ld, adapter, rows, inner, logits, ld, stream)
                             : launch<__half>(h, hidden, hidden_ld, adapter, rows, inner, logits, ld, stream);
}

} // namespace mk
