// attention_serving.cu — attention over packed sequences, one warp per (query token, query head).
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j c - m), s_j = q.k_j and
// c = scale log2 e, over the keys the mask leaves; m is the running maximum,
// and the sum and the accumulator are rescaled by 2^(m_old - m_new) when it
// grows.  A row whose mask leaves nothing is zero.  f32 arithmetic throughout.
// A warp takes 32 keys at a time: lane i forms key i's score, then every lane
// accumulates its D/32 output elements over the 32 weights.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "hs_internal.h"
#include "hs_ptx.cuh"

namespace hs {
namespace {

constexpr int kWarps = 4;

// key_ptr(j): row of key j and of its value, or null where there is none.
template <typename E, int D, typename Rows>
__device__ void attend(const E* q, E* out, int64_t n_keys, float scale_log2, const Rows& rows) {
  constexpr int kPer = D / 32;
  __shared__ float qs[kWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = lane; i < D; i += 32) qs[warp][i] = static_cast<float>(q[i]) * scale_log2;
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[kPer] = {};
  for (int64_t j0 = 0; j0 < n_keys; j0 += 32) {
    const E *k = nullptr, *v = nullptr;
    if (j0 + lane < n_keys) rows(j0 + lane, &k, &v);
    float s = -INFINITY;
    if (k) {
      s = 0.f;
#pragma unroll 4
      for (int i = 0; i < D; i += 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(k + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Elem<E>::unpack2(w[e]);
          s = fmaf(f.x, qs[warp][i + 2 * e], s);
          s = fmaf(f.y, qs[warp][i + 2 * e + 1], s);
        }
      }
    }
    float top = s;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float m_new = fmaxf(m, top);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float fix = exp2f(m - base);
    const float p = k ? exp2f(s - base) : 0.f;
    float sum = p;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * fix + sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] *= fix;
    for (int x = 0; x < 32; ++x) {
      const E* vx = reinterpret_cast<const E*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(v), x));
      const float px = __shfl_sync(0xffffffffu, p, x);
      if (!vx) continue;
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = fmaf(px, static_cast<float>(vx[lane + 32 * i]), acc[i]);
    }
    m = m_new;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[lane + 32 * i] = static_cast<E>(acc[i] * inv);
}

template <typename E, int D>
__global__ void __launch_bounds__(32 * kWarps) varlen_kernel(const VarlenIO io, float scale_log2, int* status) {
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const uint32_t token = static_cast<uint32_t>(row / io.q_heads), head = static_cast<uint32_t>(row % io.q_heads);
  if (token >= io.total_q) return;
  for (uint32_t s = 0; s < io.n_seqs; ++s) {
    const int64_t q0 = io.cu_q[s], q1 = io.cu_q[s + 1], k0 = io.cu_k[s], k1 = io.cu_k[s + 1];
    if (q0 > q1 || k0 > k1 || q0 < 0 || k0 < 0 || k1 > io.total_k || q1 > io.total_q) {
      if ((threadIdx.x & 31) == 0) atomicCAS(status, 0, static_cast<int>(kSiteBadOffsets));
      continue;
    }
    if (token < q0 || token >= q1) continue;
    const int64_t keys = io.causal ? min(k1 - k0, token - q0 + 1 + (k1 - k0) - (q1 - q0)) : k1 - k0;
    const uint32_t kv = head / (io.q_heads / io.kv_heads);
    attend<E, D>(static_cast<const E*>(io.q) + token * io.q_stride + head * D,
                 static_cast<E*>(io.out) + row * D, keys, scale_log2,
                 [&](int64_t j, const E** k, const E** v) {
                   *k = static_cast<const E*>(io.k) + (k0 + j) * io.k_stride + kv * D;
                   *v = static_cast<const E*>(io.v) + (k0 + j) * io.v_stride + kv * D;
                 });
    return;
  }
}

}  // namespace

cudaError_t launch_attention_varlen(cudaStream_t stream, int code, uint32_t d, const VarlenIO& io, float scale,
                                    int* status, uint64_t, std::string* err) {
  const uint64_t blocks = (static_cast<uint64_t>(io.total_q) * io.q_heads + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffffull) {
    if (err) *err = "too many query rows";
    return cudaErrorInvalidValue;
  }
  const float c = scale * 1.4426950408889634f;
  const dim3 g(static_cast<uint32_t>(blocks)), b(32 * kWarps);
  if (code == kBF16 && d == 64) varlen_kernel<__nv_bfloat16, 64><<<g, b, 0, stream>>>(io, c, status);
  else if (code == kBF16) varlen_kernel<__nv_bfloat16, 128><<<g, b, 0, stream>>>(io, c, status);
  else if (d == 64) varlen_kernel<__half, 64><<<g, b, 0, stream>>>(io, c, status);
  else varlen_kernel<__half, 128><<<g, b, 0, stream>>>(io, c, status);
  return cudaGetLastError();
}

}  // namespace hs
