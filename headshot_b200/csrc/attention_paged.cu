// attention_paged.cu — attention of one new token per sequence over a paged
// key-value cache, in one launch.
//
// For the g query heads that share a key head (Hq / Hkv, in tiles of 16):
//   out_h = sum_j 2^(s_hj c - m_h) v_j / sum_j 2^(s_hj c - m_h),  s_hj = q_h.k_j
// over the sequence's cached keys, c = scale log2 e.  A head tile reads every K
// and V row once (4 D bytes per key and key head) for 4 D flops per key and
// query head, so HBM bounds it; a single short sequence is bound by latency.
// Above 16 query heads per key head each further 16 read the cache again: 64
// sequences of 20,000 keys on one key head of 128, 16, 32 and 48 heads 112, 207
// and 294 us, and DRAM carries the cache three times for 48.
//
// Work is cut in tiles of 64 or 128 keys of one (sequence, key head, head tile)
// item, numbered through all items (an item has kItemCost numbers more than
// tiles, for its end).  The grid is fixed; each CTA finds the
// total from the lengths on the device and takes an equal contiguous range of
// numbers, so ragged batches and single long sequences load every SM alike and
// the host needs no lengths (a captured graph follows them).  An item that
// one CTA covers is written directly.  One that is cut leaves a partial
// (m, l, O) per CTA in the workspace; the last CTA to arrive at the item's
// counter joins them in CTA order, so results do not depend on timing, and
// returns the counter to zero.  A CTA cuts at most its first and its last
// item: two partials and one counter each, whatever the shape.
//
// Inside a CTA, each warp takes a quarter of every tile's keys through a
// ring of its own (cp.async, kStages deep, running on across items): no block
// barrier until an item ends, when the four warps' states are joined through
// the ring stage just consumed.  Scores and values go through mma.sync
// m16n8k16 with the 16 rows holding query heads: at 4 heads per key three
// quarters of the tensor work is padding, but HBM delivers a warp's keys more
// slowly than the padded products take (tcgen05's 128-row tile would
// pad 32-fold).  Rows are stored with 16-byte chunks XORed by the row's low
// bits, which makes ldmatrix free of bank conflicts.  Weights are rounded to
// the storage type for the second product, and the sum adds the rounded
// weights, so the rounding of dominant weights cancels; statistics and
// accumulators are f32.  (Weights split in two 16-bit parts, so that nothing is
// rounded away, cost 5 % at head_dim 64.)  Keys past the length are never read
// (the ring is zero-filled there).
//
// Measured in a graph of such calls: 128 sequences of 1 to 16,001 keys, 32/8 x
// 128: 165 us, 6.6 TB/s; 274,800 keys, 16 x 64: 172 us, 6.6 TB/s (a plain copy
// reaches 6.55).  Call by call, each on other caches: 184 and 192 us.  One
// sequence of 8,191 keys, 32/8 x 128: 15.9 us for 5.1 us of reading: launch 1.1,
// range 1.2, keys and values 8.3, join of the warps 0.9, partials written and
// counted 1.0, 26 of them joined 3.2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

#include "hs_internal.h"
#include "hs_ptx.cuh"

namespace hs {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;  // query heads per item
constexpr uint32_t kMaxCtas = 1024;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: weights stay below 2^8 between rescales

// 8 KB of K and V per warp and tile either way.  Head_dim 128: three stages and
// two CTAs per SM (255 registers; three CTAs of two stages spill, 1.9 times
// slower).  Head_dim 64 (200 x 1,374 keys, 16 x 64): 170 us like this (168
// registers, 44 bytes of spills), 173 us with three stages and two CTAs, 182 us
// with 16 keys per warp, four stages and three CTAs.
template <int D>
struct Shape {
  static constexpr int kWarpKeys = D == 128 ? 16 : 32;
  static constexpr int kTileKeys = kWarps * kWarpKeys;
  static constexpr int kStages = D == 128 ? 3 : 2;
  static constexpr int kCtasPerSm = D == 128 ? 2 : 3;
  static constexpr int kStageBytes = kWarpKeys * D * 2 * 2;  // K rows, then V rows; holds 16 x D f32 too
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  // An item's end costs a CTA about as much as 128 keys (query loads, the join
  // of the warps), so each item takes that many numbers more than its tiles:
  // 128 sequences of 1 to 16,001 keys, 32/8 x 128, 219 us without them, 168 us
  // with 64, 128 or 256 keys' worth.
  static constexpr uint32_t kItemCost = 128 / kTileKeys;
  // Fewest numbers per CTA.  With 128 keys' worth, 64 sequences of 100 keys
  // take 13.6 us instead of 12.6, because items that fit one CTA are cut; with
  // 512, 17.0 us.
  static constexpr uint32_t kMinTiles = 256 / kTileKeys;
};
constexpr int kMaxCtasPerSm = 3;

// Workspace: counters, then per CTA two partials of (16 x 128 O, 16 m, 16 l) f32.
constexpr size_t kCounterBytes = kMaxCtas * sizeof(uint32_t);
constexpr size_t kPartialFloats = kRows * 128 + 2 * kRows;

struct Args {
  PagedIO io;
  PagedCache c;
  uint32_t group;       // query heads per key head
  uint32_t head_tiles;  // ceil(group / 16)
  uint32_t subs;        // items per sequence: key heads x head tiles
  uint32_t ctas;        // CTAs that the GPU holds at once
  float scale_log2;
  int* status;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename E>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Elem<E>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Cached tokens of a sequence, within the block table.
__device__ __forceinline__ uint32_t seq_len(const Args& a, uint32_t s) {
  const int n = __ldg(a.c.lens + s);
  const uint32_t room = a.c.max_pages * a.c.page_size;
  if (n <= 0) return 0;
  if (static_cast<uint32_t>(n) > room) {
    atomicCAS(a.status, 0, static_cast<int>(kSiteBadLength));
    return room;
  }
  return static_cast<uint32_t>(n);
}
// An empty sequence has one tile too, which writes its zeros.
template <int D>
__device__ __forceinline__ uint32_t tiles_of(uint32_t len) {
  return len ? (len + Shape<D>::kTileKeys - 1) / Shape<D>::kTileKeys : 1;
}

// A place in the numbering of tiles: tile `tile` of item (seq, sub).
struct Place {
  unsigned long long at;  // in the numbering
  uint32_t seq, sub, tile, tiles, len;
};

template <int D>
__device__ __forceinline__ void next_tile(const Args& a, Place& p) {
  ++p.at;
  if (++p.tile < p.tiles) return;
  p.at += Shape<D>::kItemCost;
  p.tile = 0;
  if (++p.sub < a.subs) return;
  p.sub = 0;
  if (++p.seq < a.c.n_seqs) {
    p.len = seq_len(a, p.seq);
    p.tiles = tiles_of<D>(p.len);
  }
}

struct Shared {
  unsigned long long sum[kWarps];
  unsigned long long start_off;  // of the CTA's first tile inside its sequence
  uint32_t start_seq;
  uint32_t last;
  float m[kWarps][kRows];
  float l[kWarps][kRows];
};

// Sum over the block, and the exclusive prefix of this thread.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, Shared* sh, unsigned long long* excl) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();  // readers of the previous scan are done
  if (lane == 31) sh->sum[warp] = inc;
  __syncthreads();
  unsigned long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh->sum[w];
    total += sh->sum[w];
  }
  *excl = before + inc - v;
  return total;
}

// Issues this warp's keys of a tile into its ring stage.  Lane r looks up the
// cache row of key r of 16, whatever the page size, and the copies take the
// rows from the lanes (one look-up for all 16 where a page holds them gains
// nothing that is measurable: 274,800 keys, 16 x 64, 170.5 us against 171.5; 128
// ragged sequences, 32/8 x 128, 166.0 against 164.6).
template <typename E, int D>
__device__ __forceinline__ void load_tile(const Args& a, const Place& p, uint32_t stage, int warp, int lane) {
  using S = Shape<D>;
  constexpr int kChunks = D / 8;            // 16-byte chunks per row
  constexpr int kRowsPer = 32 / kChunks;    // rows one warp instruction covers
  const uint32_t key0 = p.tile * S::kTileKeys + warp * S::kWarpKeys;
  if (key0 >= p.len) return;  // the same for the whole warp
  const uint32_t chunk = lane % kChunks;
  const uint32_t head = p.sub / a.head_tiles;
  const int* table = a.c.table + static_cast<uint64_t>(p.seq) * a.c.max_pages;
  const E* kc = static_cast<const E*>(a.c.k) + 8 * chunk;
  const E* vc = static_cast<const E*>(a.c.v) + 8 * chunk;
#pragma unroll
  for (int step = 0; step < S::kWarpKeys; step += 16) {
    const uint32_t key = key0 + step + (lane & 15);
    uint64_t row = ~0ull;  // of the cache, in rows of D; all ones: no such key
    if (key < p.len) {
      const uint32_t slot = key / a.c.page_size;
      const int page = __ldg(table + slot);
      if (page < 0 || static_cast<uint32_t>(page) >= a.c.n_pages)
        atomicCAS(a.status, 0, static_cast<int>(kSiteBadPage));
      else
        row = (static_cast<uint64_t>(page) * a.c.heads + head) * a.c.page_size + (key - slot * a.c.page_size);
    }
#pragma unroll
    for (int i = 0; i < 16 / kRowsPer; ++i) {
      const uint32_t r = i * kRowsPer + lane / kChunks;  // of the step
      const uint64_t from = __shfl_sync(0xffffffffu, row, static_cast<int>(r));
      const bool ok = from != ~0ull;
      const uint64_t at = ok ? from * D : 0;
      const uint32_t dst = stage + (step + r) * (D * 2) + ((chunk ^ (r & 7)) << 4);
      cp_async16(dst, kc + at, ok);
      cp_async16(dst + S::kWarpKeys * D * 2, vc + at, ok);
    }
  }
}

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, Shape<D>::kCtasPerSm) attention_paged_kernel(const __grid_constant__ Args a) {
  using S = Shape<D>;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // The CTA's range of numbers, and the sequence it starts in.  `first` and
  // `n` are this thread's sequence of the chunk scanned last.
  auto numbers = [&](uint32_t s) -> uint32_t { return s < a.c.n_seqs ? tiles_of<D>(seq_len(a, s)) + S::kItemCost : 0u; };
  uint32_t n = numbers(tid);
  unsigned long long first;
  unsigned long long chunk = block_scan(n, &sh, &first);
  unsigned long long total = chunk;
  if (a.c.n_seqs > kThreads) {
    unsigned long long rest = 0;
    for (uint32_t s = tid + kThreads; s < a.c.n_seqs; s += kThreads) rest += numbers(s);
    unsigned long long unused;
    total += block_scan(rest, &sh, &unused);
  }
  // No more CTAs than have kMinTiles tiles each: 8,191 keys, 32/8 x 128, 15.9 us
  // with 208 CTAs and items cut in 26, 16.4 us with 260 and items cut in 33.
  const unsigned long long tiles = (total - static_cast<unsigned long long>(a.c.n_seqs) * S::kItemCost) * a.subs;
  const unsigned long long some = (tiles + S::kMinTiles - 1) / S::kMinTiles;
  const unsigned long long ctas = some < a.ctas ? some : a.ctas;
  total *= a.subs;
  const unsigned long long even = (total + ctas - 1) / ctas;
  const unsigned long long per = even < S::kMinTiles ? S::kMinTiles : even;
  const unsigned long long start = blockIdx.x * per;
  if (start >= total) return;
  const unsigned long long end = start + per < total ? start + per : total;
  unsigned long long base = 0;
  uint32_t s0 = 0;
  while ((base + chunk) * a.subs <= start) {
    base += chunk;
    s0 += kThreads;
    if (s0 >= a.c.n_seqs) return;
    n = numbers(s0 + tid);
    chunk = block_scan(n, &sh, &first);
  }
  first = (base + first) * a.subs;
  if (first <= start && start < first + static_cast<unsigned long long>(n) * a.subs) {
    sh.start_seq = s0 + tid;
    sh.start_off = start - first;
  }
  __syncthreads();
  Place cur;
  cur.seq = sh.start_seq;
  cur.len = seq_len(a, cur.seq);
  cur.tiles = tiles_of<D>(cur.len);
  cur.sub = static_cast<uint32_t>(sh.start_off / (cur.tiles + S::kItemCost));
  cur.tile = static_cast<uint32_t>(sh.start_off % (cur.tiles + S::kItemCost));
  cur.at = start;
  if (cur.tile >= cur.tiles) {  // starts among an item's extra numbers: on to the next item
    cur.at -= cur.tile - (cur.tiles - 1);
    cur.tile = cur.tiles - 1;
    next_tile<D>(a, cur);
  }

  const uint32_t my_ring = smem_u32(ring) + warp * S::kStages * S::kStageBytes;
  Place ahead = cur;
  uint32_t load_stage = 0;
  auto load_next = [&] {
    if (ahead.at < end) {
      load_tile<E, D>(a, ahead, my_ring + load_stage * S::kStageBytes, warp, lane);
      next_tile<D>(a, ahead);
    }
    load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) load_next();

  uint32_t q[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];                   // m: running maximum of the scores, before the scale
  const float threshold = fminf(kRescaleThreshold / a.scale_log2, 1e30f);  // finite: -inf + it stays below any score
  const uint32_t row_lo = lane >> 2;  // rows row_lo and row_lo + 8 of the head tile

  bool fresh = true;                  // the next tile starts a segment
  for (uint32_t st = 0; cur.at < end; st = st + 1 == S::kStages ? 0 : st + 1) {
    const uint32_t head = cur.sub / a.head_tiles;
    const uint32_t row0 = (cur.sub % a.head_tiles) * kRows;
    const uint32_t rows = min(static_cast<uint32_t>(kRows), a.group - row0);
    if (fresh) {
      fresh = false;
      const E* qs = static_cast<const E*>(a.io.q) + cur.seq * a.io.q_stride +
                    static_cast<uint64_t>(head * a.group + row0) * D + 2 * (lane & 3);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t r = row_lo + (x & 1) * 8;
          q[k][x] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(qs + r * D + k * 16 + (x >> 1) * 8)) : 0u;
        }
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][x] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    cp_async_wait<S::kStages - 2>();
    __syncwarp();
    load_next();
    const uint32_t stage = my_ring + st * S::kStageBytes;
    const uint32_t key0 = cur.tile * S::kTileKeys + warp * S::kWarpKeys;
    if (key0 < cur.len) {
      // Scores: rows = heads, 8-key column tiles.
      constexpr int kCols = S::kWarpKeys / 8;
      float s[kCols][4] = {};
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int t = 0; t < kCols; t += 2) {
          uint32_t b[4];
          const uint32_t r = 8 * t + (lane & 7) + ((lane >> 4) << 3), ch = 2 * k + ((lane >> 3) & 1);
          ldsm4(b, stage + r * (D * 2) + ((ch ^ (r & 7)) << 4));
          mma16816<E>(s[t], q[k], b[0], b[1]);
          mma16816<E>(s[t + 1], q[k], b[2], b[3]);
        }
      const uint32_t valid = cur.len - key0;
      if (valid < S::kWarpKeys) {
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (t * 8 + 2 * (lane & 3) + (x & 1) >= valid) s[t][x] = -INFINITY;
      }
      float top[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
        for (int x = 1; x < kCols; ++x) t = fmaxf(t, fmaxf(s[x][2 * h], s[x][2 * h + 1]));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        top[h] = t;
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] + threshold || top[1] > m[1] + threshold)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float m_new = fmaxf(m[h], top[h]);
          const float f = m_new == -INFINITY ? 1.f : ex2_approx((m[h] - m_new) * a.scale_log2);
          m[h] = m_new;
          l[h] *= f;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * h] *= f;
            o[n][2 * h + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int g = 0; g < kCols; g += 2) {  // 16 keys
        uint32_t p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float base_m = m[h] == -INFINITY ? 0.f : m[h];
            const uint32_t w = Elem<E>::pack2(ex2_approx((s[g + t][2 * h] - base_m) * a.scale_log2),
                                              ex2_approx((s[g + t][2 * h + 1] - base_m) * a.scale_log2));
            const float2 f = Elem<E>::unpack2(w);
            l[h] += f.x + f.y;
            p[2 * t + h] = w;
          }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];
          const uint32_t r = 8 * g + (lane & 7) + (((lane >> 3) & 1) << 3), ch = 2 * n + (lane >> 4);
          ldsm4_t(b, stage + S::kWarpKeys * D * 2 + r * (D * 2) + ((ch ^ (r & 7)) << 4));
          mma16816<E>(o[2 * n], p, b[0], b[1]);
          mma16816<E>(o[2 * n + 1], p, b[2], b[3]);
        }
      }
    }

    const bool item_ends = cur.tile + 1 == cur.tiles;
    if (item_ends || cur.at + 1 == end) {
      // Join the warps: states through the stage this tile came from (its next
      // load is issued one iteration on, behind the block barrier below).
      __syncwarp();
      float* dump = reinterpret_cast<float*>(ring + (warp * S::kStages + st) * S::kStageBytes);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = row_lo + 8 * h;
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if ((lane & 3) == 0) {
          sh.m[warp][r] = m[h];
          sh.l[warp][r] = l[h];
        }
        if (r < rows) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const uint32_t col = (8 * n + 2 * (lane & 3)) ^ ((r & 3) << 3);
            *reinterpret_cast<float2*>(dump + r * D + col) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
          }
        }
      }
      __syncthreads();
      const unsigned long long item0 = cur.at - cur.tile;  // first tile of the item
      const unsigned long long item1 = item0 + cur.tiles;
      const uint32_t cta0 = static_cast<uint32_t>(item0 / per), cta1 = static_cast<uint32_t>((item1 - 1) / per);
      const bool whole = cta0 == cta1;
      E* out = static_cast<E*>(a.io.out) +
               (static_cast<uint64_t>(cur.seq) * a.io.q_heads + head * a.group + row0) * D;
      uint32_t* counters = static_cast<uint32_t*>(a.io.workspace);
      float* partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a.io.workspace) + kCounterBytes);
      auto partial = [&](uint32_t cta) { return partials + (2 * static_cast<size_t>(cta) + (cta == cta0)) * kPartialFloats; };
      float* mine = partial(blockIdx.x);
      for (uint32_t e = tid; e < rows * (D / 4); e += kThreads) {
        const uint32_t r = e / (D / 4), c4 = (e % (D / 4)) * 4;
        float mt = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sh.m[w][r]);
        float lt = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = sh.m[w][r] == -INFINITY ? 0.f : ex2_approx((sh.m[w][r] - mt) * a.scale_log2);
          lt = fmaf(sh.l[w][r], f, lt);
          const float4 v = *reinterpret_cast<const float4*>(
              ring + (w * S::kStages + st) * S::kStageBytes +
              (r * D + (c4 ^ ((r & 3) << 3))) * 4);
          acc.x = fmaf(v.x, f, acc.x);
          acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z);
          acc.w = fmaf(v.w, f, acc.w);
        }
        if (whole) {
          const float inv = lt == 0.f ? 0.f : 1.f / lt;
          *reinterpret_cast<uint2*>(out + r * D + c4) =
              make_uint2(Elem<E>::pack2(acc.x * inv, acc.y * inv), Elem<E>::pack2(acc.z * inv, acc.w * inv));
        } else {
          *reinterpret_cast<float4*>(mine + r * D + c4) = acc;
          if (c4 == 0) {
            mine[kRows * D + r] = mt;
            mine[kRows * D + kRows + r] = lt;
          }
        }
      }
      if (!whole) {
        __threadfence();
        __syncthreads();
        if (tid == 0) sh.last = atomicAdd(counters + cta0, 1u) == cta1 - cta0;
        __syncthreads();
        if (sh.last) {
          __threadfence();
          for (uint32_t e = tid; e < rows * (D / 4); e += kThreads) {
            const uint32_t r = e / (D / 4), c4 = (e % (D / 4)) * 4;
            // In batches whose loads are all in flight together.
            constexpr uint32_t kPart = 16;
            float mt = -INFINITY, lt = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t c0 = cta0; c0 <= cta1; c0 += kPart) {
              float mc[kPart], lc[kPart];
              float4 v[kPart];
#pragma unroll
              for (uint32_t x = 0; x < kPart; ++x) {
                const bool have = c0 + x <= cta1;
                const float* src = partial(c0 + x);
                mc[x] = have ? __ldcg(src + kRows * D + r) : -INFINITY;
                lc[x] = have ? __ldcg(src + kRows * D + kRows + r) : 0.f;
                v[x] = have ? __ldcg(reinterpret_cast<const float4*>(src + r * D + c4)) : make_float4(0.f, 0.f, 0.f, 0.f);
              }
              float m_new = mt;
#pragma unroll
              for (uint32_t x = 0; x < kPart; ++x) m_new = fmaxf(m_new, mc[x]);
              const float f0 = mt == -INFINITY ? 0.f : ex2_approx((mt - m_new) * a.scale_log2);
              mt = m_new;
              lt *= f0;
              acc.x *= f0;
              acc.y *= f0;
              acc.z *= f0;
              acc.w *= f0;
#pragma unroll
              for (uint32_t x = 0; x < kPart; ++x) {
                const float f = mc[x] == -INFINITY ? 0.f : ex2_approx((mc[x] - mt) * a.scale_log2);
                lt = fmaf(lc[x], f, lt);
                acc.x = fmaf(v[x].x, f, acc.x);
                acc.y = fmaf(v[x].y, f, acc.y);
                acc.z = fmaf(v[x].z, f, acc.z);
                acc.w = fmaf(v[x].w, f, acc.w);
              }
            }
            const float inv = lt == 0.f ? 0.f : 1.f / lt;
            *reinterpret_cast<uint2*>(out + r * D + c4) =
                make_uint2(Elem<E>::pack2(acc.x * inv, acc.y * inv), Elem<E>::pack2(acc.z * inv, acc.w * inv));
          }
          if (tid == 0) atomicExch(counters + cta0, 0u);
        }
      }
      __syncthreads();  // the stage and sh may be written again
      fresh = true;
    }
    next_tile<D>(a, cur);
  }
  cp_async_wait<0>();
}

template <typename E, int D>
cudaError_t launch(cudaStream_t stream, Args& a) {
  using S = Shape<D>;
  const void* f = reinterpret_cast<const void*>(attention_paged_kernel<E, D>);
  const cudaError_t e = ensure_dynamic_smem(f, S::kSmem);
  if (e != cudaSuccess) return e;
  uint64_t ctas = static_cast<uint64_t>(current_sm_count()) * S::kCtasPerSm;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  // The split follows this number and the lengths, which only the kernel knows;
  // the launch leaves out the CTAs that get nothing even if every length fills
  // the block table.
  a.ctas = static_cast<uint32_t>(ctas);
  const uint64_t most = (static_cast<uint64_t>(a.c.max_pages) * a.c.page_size + S::kTileKeys - 1) / S::kTileKeys;
  const uint64_t tiles = static_cast<uint64_t>(a.c.n_seqs) * a.subs * (most ? most : 1);
  ctas = std::min<uint64_t>(ctas, (tiles + S::kMinTiles - 1) / S::kMinTiles);
  attention_paged_kernel<E, D><<<static_cast<uint32_t>(ctas), kThreads, S::kSmem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

size_t attention_paged_workspace_bytes() {
  uint64_t ctas = static_cast<uint64_t>(current_sm_count()) * kMaxCtasPerSm;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  return kCounterBytes + ctas * 2 * kPartialFloats * sizeof(float);
}

cudaError_t launch_attention_paged(cudaStream_t stream, int code, uint32_t d, const PagedIO& io, const PagedCache& c,
                                   float scale, int* status) {
  Args a;
  a.io = io;
  a.c = c;
  a.group = io.q_heads / c.heads;
  a.head_tiles = (a.group + kRows - 1) / kRows;
  a.subs = c.heads * a.head_tiles;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status;
  if (code == kBF16)
    return d == 64 ? launch<__nv_bfloat16, 64>(stream, a) : launch<__nv_bfloat16, 128>(stream, a);
  return d == 64 ? launch<__half, 64>(stream, a) : launch<__half, 128>(stream, a);
}

}  // namespace hs
