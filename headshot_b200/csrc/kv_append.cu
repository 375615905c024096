// kv_append.cu — new tokens' keys and values into a paged cache, with the
// position rotation (rotate-half RoPE as rope_apply, src/engine/ops.rs:202-223)
// applied to the keys, and to the queries of the same tokens, on the way.
//
// Token i of sequence s sits at position p = lens[s] - n_new(s) + i, where
// lens counts the sequence's tokens after the append.  For element e < D/2:
//   y[e]       = x[e] cos[r][e] - x[e + D/2] sin[r][e]
//   y[e + D/2] = x[e + D/2] cos[r][e + D/2] + x[e] sin[r][e + D/2]
// in f32, rounded once, with table row r = p (mod tokens_per_frame) - prefix;
// r < 0 passes through.  Every element is read and written once, so the
// kernel is bound by HBM for prompts and by launch latency for single tokens.
//
// One thread owns a (token, chunk): elements [8c, 8c + 8) and their rotation
// partners [D/2 + 8c, +8).  It loads the chunk's 32 table values once and then
// takes every lane-th head of the token with them, kBatch heads' loads in
// flight before the first store, so a head row costs two 16-byte loads and
// two 16-byte stores and the table stays out of the loop.  The first heads'
// loads are issued before the token's place (sequence, length, page, table row)
// is looked up, so the four dependent reads hide behind them.  An element is
// read and written by the same thread, so q_out may be q and k_out may be k.
//
// Measured: 32,768 tokens, 32/8 x 128: 139 us, 6.5 TB/s (a plain copy reaches
// 6.55); 24 ragged prompts of 8,898 tokens 41.6 us, 5.8 TB/s; one token 2.7 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hs_internal.h"
#include "hs_ptx.cuh"

namespace hs {
namespace {

// 40 prompts of 10 to 1,500 tokens, 16/16 x 64 and 16/16 x 128: 128 threads with
// 2, 4, 6 heads in flight 29.2, 30.0, 31.0 and 52.7, 52.3, 52.4 us; 256 threads
// with 4 33.7 and 53.6; 64 threads like 128, but slower for single tokens.
constexpr int kThreads = 128;
constexpr int kBatch = 4;  // heads in flight per thread

struct Args {
  KvAppend a;
  PagedCache c;
  int* status;
};

// Largest s in [0, n) with cu[s] <= t, by 32-way steps of a whole warp.
__device__ __forceinline__ uint32_t find_seq(const int* cu, uint32_t n, int t) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t lo = 0, len = n;
  while (len > 1) {
    const uint32_t step = (len + 31) / 32;
    const uint32_t at = lo + lane * step;
    const bool below = lane * step < len && __ldg(cu + at) <= t;
    const uint32_t votes = __ballot_sync(0xffffffffu, below);
    const uint32_t last = votes ? 31 - __clz(votes) : 0;
    const uint32_t end = lo + len;
    lo += last * step;
    len = min(step, end - lo);
  }
  return lo;
}

// D/16 threads of 8 + 8 elements per head row, `lanes` head rows side by side,
// kThreads / (D/16 * lanes) tokens per block.
template <typename E, int D>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ Args args, uint32_t lanes) {
  constexpr uint32_t kChunks = D / 16;
  const KvAppend& a = args.a;
  const PagedCache& c = args.c;
  const uint32_t per_token = kChunks * lanes;  // a multiple of 32: a warp holds one token
  const uint32_t tokens = kThreads / per_token;
  const uint32_t token = blockIdx.x * tokens + threadIdx.x / per_token;
  // A token sees the offsets of its own sequence only, so the grid shares out
  // the neighbouring pairs, one a thread, to find the falling ones.
  if (a.cu_new) {
    for (uint64_t s = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x; s < c.n_seqs;
         s += static_cast<uint64_t>(gridDim.x) * kThreads)
      if (__ldg(a.cu_new + s + 1) < __ldg(a.cu_new + s)) atomicCAS(args.status, 0, static_cast<int>(kSiteBadOffsets));
  }
  if (token >= a.n_tokens) return;
  const uint32_t in_token = threadIdx.x % per_token;
  const uint32_t chunk = in_token % kChunks;
  const uint32_t lane = in_token / kChunks;

  const uint32_t q_rows = a.q ? a.q_heads : 0;
  const uint32_t rows = q_rows + 2 * c.heads;
  const E* qt = static_cast<const E*>(a.q) + token * a.q_stride;
  const E* kt = static_cast<const E*>(a.k) + token * a.k_stride;
  const E* vt = static_cast<const E*>(a.v) + token * a.v_stride;
  uint4 lo[kBatch], hi[kBatch];
  auto load = [&](uint32_t r0) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const uint32_t r = r0 + b * lanes;
      if (r >= rows) break;
      const E* src = r < q_rows             ? qt + static_cast<uint64_t>(r) * D
                     : r < q_rows + c.heads ? kt + static_cast<uint64_t>(r - q_rows) * D
                                            : vt + static_cast<uint64_t>(r - q_rows - c.heads) * D;
      lo[b] = *reinterpret_cast<const uint4*>(src + 8 * chunk);
      hi[b] = *reinterpret_cast<const uint4*>(src + D / 2 + 8 * chunk);
    }
  };
  load(lane);  // in flight while the token's place is looked up: four dependent reads

  uint32_t seq = token;
  int64_t pos;
  if (a.cu_new) {
    const int64_t start = __ldg(a.cu_new), last = __ldg(a.cu_new + c.n_seqs);
    const bool fits = start == 0 && last <= static_cast<int64_t>(a.n_tokens);
    if (!fits && in_token == 0) atomicCAS(args.status, 0, static_cast<int>(kSiteBadOffsets));
    if (token >= last || token < start) return;
    seq = find_seq(a.cu_new, c.n_seqs, static_cast<int>(token));
    const int64_t first = __ldg(a.cu_new + seq), end = __ldg(a.cu_new + seq + 1);
    // An end past the rows or past the last offset would count the token's
    // position back from tokens that do not exist.
    if (first < 0 || token < first || token >= end || end > last || end > static_cast<int64_t>(a.n_tokens)) {
      if (in_token == 0) atomicCAS(args.status, 0, static_cast<int>(kSiteBadOffsets));
      return;
    }
    pos = static_cast<int64_t>(__ldg(c.lens + seq)) - (end - token);
  } else {
    pos = static_cast<int64_t>(__ldg(c.lens + seq)) - 1;
  }
  if (pos < 0) return;  // padding
  const uint32_t p = static_cast<uint32_t>(pos);

  // Cache row and rotation row of the token; a bad index skips the token.
  const uint32_t slot = p / c.page_size;
  int bad = 0;
  uint64_t cache_row = 0;  // of head 0, in rows of D
  if (slot >= c.max_pages) {
    bad = kSiteBadLength;
  } else {
    const int page = __ldg(c.table + static_cast<uint64_t>(seq) * c.max_pages + slot);
    if (page < 0 || static_cast<uint32_t>(page) >= c.n_pages) bad = kSiteBadPage;
    cache_row = static_cast<uint64_t>(page) * c.heads * c.page_size + p % c.page_size;
  }
  bool rotate = false;
  uint64_t table_at = 0;
  if (a.sin_t) {
    const uint32_t f = a.tokens_per_frame ? p % a.tokens_per_frame : p;
    rotate = f >= a.prefix;
    if (rotate) {
      if (f - a.prefix >= a.rope_rows) bad = kSiteBadRopeRow;
      table_at = static_cast<uint64_t>(f - a.prefix) * D + 8 * chunk;
    }
  }
  if (bad) {
    if (in_token == 0) atomicCAS(args.status, 0, bad);
    return;
  }

  float sin_v[16], cos_v[16];  // [0, 8): lower half's, [8, 16): upper half's
  if (rotate) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t at = table_at + (i >> 1) * (D / 2) + (i & 1) * 4;
      *reinterpret_cast<float4*>(sin_v + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at));
      *reinterpret_cast<float4*>(cos_v + 4 * i) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at));
    }
  }

  for (uint32_t r0 = lane; r0 < rows;) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const uint32_t r = r0 + b * lanes;
      if (r >= rows) break;
      const bool is_v = r >= q_rows + c.heads;
      if (rotate && !is_v) {
        uint32_t* l = reinterpret_cast<uint32_t*>(&lo[b]);
        uint32_t* h = reinterpret_cast<uint32_t*>(&hi[b]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = Elem<E>::unpack2(l[i]), y = Elem<E>::unpack2(h[i]);
          l[i] = Elem<E>::pack2(x.x * cos_v[2 * i] - y.x * sin_v[2 * i],
                                x.y * cos_v[2 * i + 1] - y.y * sin_v[2 * i + 1]);
          h[i] = Elem<E>::pack2(y.x * cos_v[8 + 2 * i] + x.x * sin_v[8 + 2 * i],
                                y.y * cos_v[8 + 2 * i + 1] + x.y * sin_v[8 + 2 * i + 1]);
        }
      }
      auto put = [&](E* dst) {
        *reinterpret_cast<uint4*>(dst + 8 * chunk) = lo[b];
        *reinterpret_cast<uint4*>(dst + D / 2 + 8 * chunk) = hi[b];
      };
      if (r < q_rows) {
        put(static_cast<E*>(a.q_out) + (static_cast<uint64_t>(token) * a.q_heads + r) * D);
      } else {
        const uint32_t h = is_v ? r - q_rows - c.heads : r - q_rows;
        E* cache = static_cast<E*>(is_v ? c.v : c.k);
        put(cache + (cache_row + static_cast<uint64_t>(h) * c.page_size) * D);
        if (!is_v && a.k_out) put(static_cast<E*>(a.k_out) + (static_cast<uint64_t>(token) * c.heads + h) * D);
      }
    }
    r0 += kBatch * lanes;
    load(r0);
  }
}

template <typename E, int D>
cudaError_t run(cudaStream_t stream, const Args& args) {
  // Few tokens: all of a block's threads on one token's heads; many tokens:
  // as few head lanes as make whole warps, so a thread reuses its table
  // values most.
  constexpr uint32_t chunks = D / 16;
  const uint32_t lanes = args.a.n_tokens <= static_cast<uint32_t>(current_sm_count()) ? kThreads / chunks : 32 / chunks;
  const uint32_t tokens = kThreads / (chunks * lanes);
  kv_append_kernel<E, D><<<(args.a.n_tokens + tokens - 1) / tokens, kThreads, 0, stream>>>(args, lanes);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_append(cudaStream_t stream, int code, uint32_t d, const KvAppend& a, const PagedCache& c,
                             int* status) {
  if (a.n_tokens == 0 || c.n_seqs == 0) return cudaSuccess;
  const Args args{a, c, status};
  if (code == kBF16)
    return d == 64 ? run<__nv_bfloat16, 64>(stream, args) : run<__nv_bfloat16, 128>(stream, args);
  return d == 64 ? run<__half, 64>(stream, args) : run<__half, 128>(stream, args);
}

}  // namespace hs
