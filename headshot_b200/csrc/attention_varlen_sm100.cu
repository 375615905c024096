// attention_varlen_sm100.cu — flash attention over packed sequences on
// tcgen05: causal or not, grouped heads, head_dim 64 and 128, f16 / bf16.
//
//   out_i = sum_j 2^(s_ij c - m_i) v_j / sum_j 2^(s_ij c - m_i),
//   s_ij = q_i.k_j over the keys the mask leaves, c = scale log2 e.
//
// The CTA is laid out as attn_fwd_sm100's (attention_sm100.cu): two softmax
// warpgroups of 128 query rows, one MMA warp each, a TMA producer warp, two
// score buffers per warpgroup in TMEM so that S(j+1) is ready while S(j) turns
// into P(j), P written over the scores it came from and read from TMEM by the
// PV product.  What packing, masks and grouped heads change:
//
// - A 128-row tile holds the g = Hq / Hkv heads of floor(128 / g) tokens, token
//   by token (one TMA box), so all heads that share keys share the K/V tiles
//   and a short sequence fills rows with heads.  An item is two such tiles of
//   one (sequence, key head) against its keys.
// - The grid covers every item the packed rows can hold; a resident CTA takes
//   over the next pending one with clusterlaunchcontrol.try_cancel while it
//   works on the current one.  Scheduling is dynamic without a counter in
//   memory, so launches share nothing.  Which sequence an item belongs to is
//   found from the offsets on the device.  Items of a (sequence, key head) go
//   out longest first, head by head, so the CTAs at work share K/V in L2.
// - Under a causal mask each warpgroup stops at its own last key tile; tiles
//   that cross the diagonal or the sequence's end are masked element by element.
// - The keys of a tile that lie behind the sequence belong to the next one:
//   their scores are masked, and their values, which the PV product would
//   still multiply by zero, are overwritten with zeros in shared memory, so
//   infinities or NaN there cannot reach the result.
//
// Head_dim 64: 96-key tiles; 128: 64-key tiles, since two f32 accumulators of
// 128 columns leave 256 of TMEM's 512 columns for the four score buffers.
// Rounding: P is rounded to the storage type for the PV product and the row sum
// adds the rounded P; statistics and accumulators are f32.
#include <cuda.h>

#include <algorithm>

#include "hs_internal.h"
#include "hs_ptx.cuh"

namespace hs {
namespace {

constexpr int kBM = 128;  // query rows per tile / softmax warpgroup
constexpr int kItemSlots = 4;
constexpr int kItemReaders = 8 + 2;
constexpr int kThreads = 384;
constexpr uint32_t kLaunchRegs = 168;  // 65536 / 384 rounded down to a multiple of 8
constexpr uint32_t kSoftmaxRegs = 224;
constexpr uint32_t kControlRegs = 56;
static_assert(2 * kSoftmaxRegs + kControlRegs <= 3 * kLaunchRegs, "setmaxnreg split exceeds the launch budget");
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp0 = 9;
constexpr int kTmemWarp = 11;
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: p <= 2^8 between rescales

template <int D>
struct Shape {
  static constexpr int kBN = D == 64 ? 96 : 64;
  static constexpr int kPairs = kBN / 2;
  static constexpr int kStages = D == 64 ? 6 : 5;
  static constexpr int kQBufs = D == 64 ? 2 : 1;
  static constexpr int kHalves = D / 64;             // 128-byte column blocks of a row
  static constexpr int kQTileBytes = kBM * D * 2;
  static constexpr int kKvTileBytes = kBN * D * 2;
  static constexpr uint32_t kQHalf = kBM * 128;      // bytes from one column block to the next
  static constexpr uint32_t kKvHalf = kBN * 128;
  static constexpr int kEmuPer8 = 2;  // of every 8 exponential pairs, this many run on the FMA pipe
  __host__ __device__ static constexpr uint32_t col_s(int wg, int buf) { return static_cast<uint32_t>((2 * wg + buf) * kBN); }
  __host__ __device__ static constexpr uint32_t col_o(int wg) { return static_cast<uint32_t>(4 * kBN + D * wg); }
  static_assert(4 * kBN + 2 * D <= 512, "TMEM budget");
  static_assert(kKvHalf % 1024 == 0, "swizzle atoms stay 1024-byte aligned");
};

enum : int {
  kSiteQFull = 0x301,
  kSiteKvFull = 0x302,
  kSiteQEmpty = 0x303,
  kSitePFull = 0x304,
  kSiteSFull = 0x305,
  kSiteODone = 0x306,
  kSiteKvEmpty = 0x307,
  kSiteItemFull = 0x308,
  kSiteItemEmpty = 0x309,
  kSiteNext = 0x30a,
};

// One unit of work, as the producer decodes it.
struct Item {
  int q_row;     // first query token of the item, in the packed rows; kNoItem: no more work
  int tokens;    // query tokens from there to the sequence's end (may exceed the item)
  int k_row;     // the sequence's first key
  int n_keys;    // its keys
  int lim;       // last key the item's first token sees (negative: none)
  uint32_t head; // key head
  uint32_t n;    // key tiles of the item: the larger of its two warpgroups'
};
constexpr int kNoItem = -1;

// Barrier phases are counted per barrier across all items of a CTA, as in
// attn_fwd_sm100: when a waiter asks for completion k, completion k-1 has
// already happened and completion k+1 needs an action the waiter takes
// after this wait.  Tile counts differ from item to item and between the
// warpgroups, so each role keeps its own counts.
template <int D>
struct Ctrl {
  using S = Shape<D>;
  uint64_t kv_full[S::kStages];
  uint64_t kv_empty[S::kStages];
  uint64_t q_full[2][S::kQBufs];
  uint64_t q_empty[2][S::kQBufs];
  uint64_t s_full[2][2];
  uint64_t p_full[2][2];
  uint64_t pv_prev[2];
  uint64_t pv_last[2];
  uint64_t drain[2];
  uint64_t item_full[kItemSlots];
  uint64_t item_empty[kItemSlots];
  uint64_t next_full;
  uint4 next;  // try_cancel's answer
  Item item[kItemSlots];
  uint32_t tmem_base;
  int abort_flag;
};

template <int D>
constexpr size_t smem_bytes() {
  using S = Shape<D>;
  return 1024 + 2 * S::kQBufs * S::kQTileBytes + 2 * S::kStages * S::kKvTileBytes + sizeof(Ctrl<D>);
}
static_assert(smem_bytes<64>() <= 232448 && smem_bytes<128>() <= 232448, "shared memory per CTA");

struct Args {
  void* out;
  const int* cu_q;
  const int* cu_k;
  uint32_t n_seqs, total_q, total_k;
  uint32_t group;        // query heads per key head
  uint32_t kv_heads;
  uint32_t tile_tokens;  // tokens per 128-row tile: 128 / group
  int causal;
  float scale_log2;
  int* status;
  uint64_t timeout_ns;
};

__device__ __forceinline__ float u2f(uint32_t u) { return __uint_as_float(u); }

template <int kStages>
struct RingPos {
  uint32_t stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status,
                                          int site, uint64_t timeout_ns) {
  const bool r = mbar_wait(bar, parity, abort_flag, status, site, timeout_ns);
  return __all_sync(0xffffffffu, r);
}

__device__ __forceinline__ void mbar_arrive_elect(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

// Next item for a reader warp (all lanes), from slot k % kItemSlots.
template <int D>
__device__ __forceinline__ bool next_item(const Args& a, Ctrl<D>* ctl, uint32_t k, Item* item) {
  const uint32_t slot = k % kItemSlots;
  if (!warp_wait(&ctl->item_full[slot], (k / kItemSlots) & 1, &ctl->abort_flag, a.status, kSiteItemFull,
                 a.timeout_ns))
    return false;
  const volatile Item* src = &ctl->item[slot];
  item->q_row = src->q_row;
  item->tokens = src->tokens;
  item->k_row = src->k_row;
  item->n_keys = src->n_keys;
  item->lim = src->lim;
  item->head = src->head;
  item->n = src->n;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&ctl->item_empty[slot]);
  return true;
}

// Key tiles of warpgroup wg's rows: up to the last key its last token sees.
template <int D>
__device__ __forceinline__ uint32_t wg_tiles(const Args& a, const Item& it, int wg) {
  const int first = wg * static_cast<int>(a.tile_tokens);
  if (first >= it.tokens) return 0;
  int keys = it.n_keys;
  if (a.causal) keys = min(keys, it.lim + min(first + static_cast<int>(a.tile_tokens), it.tokens));
  return keys > 0 ? static_cast<uint32_t>(keys + Shape<D>::kBN - 1) / Shape<D>::kBN : 0u;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair on the FMA pipe: the same reduction and cubic as
// attn_fwd_sm100's (max relative error 8.3e-5, inputs clamped at -125).
constexpr float kExpMagic = 12582912.0f;  // 1.5 * 2^23
constexpr float kExpC0 = 0.99991959f;
constexpr float kExpC1 = 0.69326216f;
constexpr float kExpC2 = 0.24271429f;
constexpr float kExpC3 = 0.05521307f;

__device__ __forceinline__ void exp2_poly2(float x0, float x1, float& y0, float& y1) {
  x0 = fmaxf(x0, -125.f);
  x1 = fmaxf(x1, -125.f);
  float t0, t1, r0, r1, f0, f1, p0, p1;
  add2(t0, t1, x0, x1, kExpMagic, kExpMagic);
  add2(r0, r1, t0, t1, -kExpMagic, -kExpMagic);
  fma2(f0, f1, r0, r1, -1.f, -1.f, x0, x1);
  fma2(p0, p1, f0, f1, kExpC3, kExpC3, kExpC2, kExpC2);
  fma2(p0, p1, p0, p1, f0, f1, kExpC1, kExpC1);
  fma2(p0, p1, p0, p1, f0, f1, kExpC0, kExpC0);
  y0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  y1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

template <typename E, int D>
__device__ void softmax_role(const Args& a, Ctrl<D>* ctl, uint32_t tmem, int warp, int lane) {
  using S = Shape<D>;
  constexpr int kBN = S::kBN;
  const int wg = warp >> 2;
  const int wq = warp & 3;
  const uint32_t row = static_cast<uint32_t>(wq * 32 + lane);
  volatile int* abort_flag = &ctl->abort_flag;
  const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
  const uint32_t tO = tmem + lane_base + S::col_o(wg);
  const float c = a.scale_log2;
  // The row's token within the tile and head within the group.
  const uint32_t tok = row / a.group, head = row - tok * a.group;
  const bool in_tile = tok < a.tile_tokens;
  const uint32_t row_elems = a.group * a.kv_heads * D;
  // Completions seen before the item: bits of s_full[0], s_full[1], pv_last,
  // pv_prev parities.
  uint32_t base_bits = 0;
  auto s_parity = [&](uint32_t t) { return ((base_bits >> (t & 1)) + (t >> 1)) & 1; };

  Item nxt{};
  bool have_nxt = false;
  for (uint32_t k = 0;; ++k) {
    Item it;
    if (have_nxt) {
      it = nxt;
      have_nxt = false;
    } else if (!next_item<D>(a, ctl, k, &it)) {
      return;
    }
    if (it.q_row == kNoItem) break;
    const int token = wg * static_cast<int>(a.tile_tokens) + static_cast<int>(tok);
    if (wg * static_cast<int>(a.tile_tokens) >= it.tokens) continue;
    const uint32_t n = wg_tiles<D>(a, it, wg);
    const bool valid = in_tile && token < it.tokens;
    const int lim = a.causal ? min(it.lim + token, it.n_keys - 1) : it.n_keys - 1;  // last key the row sees
    // Rows of a warp see more keys the later their token: its first row's limit is the lowest.
    const int lim_warp = __shfl_sync(0xffffffffu, lim, 0);
    E* out = static_cast<E*>(a.out) + static_cast<uint64_t>(it.q_row + token) * row_elems +
             (it.head * a.group + head) * D;

    float m_run = -INFINITY, l = 0.f;
    for (uint32_t j = 0; j < n; ++j) {
      const int b = static_cast<int>(j & 1);
      if (!warp_wait(&ctl->s_full[wg][b], s_parity(j), abort_flag, a.status, kSiteSFull, a.timeout_ns)) return;
      tc_fence_after();
      const uint32_t tS = tmem + lane_base + S::col_s(wg, b);
      uint32_t s[kBN];
#pragma unroll
      for (int x = 0; x < kBN; x += 32) tmem_ld32(tS + x, s + x);
      tmem_wait_ld_regs<kBN>(s);
      const int kb = static_cast<int>(j) * kBN;
      if (kb + kBN - 1 > lim_warp) {
        const int left = lim - kb;
#pragma unroll
        for (int i = 0; i < kBN; ++i)
          if (i > left) s[i] = __float_as_uint(-INFINITY);
      }
      float factor = 1.f;
      bool need = false;
      float m4[4] = {u2f(s[0]), u2f(s[1]), u2f(s[2]), u2f(s[3])};
#pragma unroll
      for (int i = 4; i < kBN; i += 2) m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], u2f(s[i]), u2f(s[i + 1]));
      const float m_tile = max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]) * c;
      if (j == 0) {
        m_run = m_tile;
      } else if (m_tile > m_run + kRescaleThreshold) {
        factor = ex2_approx(m_run - m_tile);
        m_run = m_tile;
        l *= factor;
        need = true;
      }
      // A row that sees no key has m_run = -inf and turns into NaN here: its
      // output is set to zero below, and no other row reads it.
      const float neg_m = -m_run;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t pk[S::kPairs];
#pragma unroll
      for (int i = 0; i < S::kPairs; ++i) {
        float x0, x1, p0, p1;
        fma2(x0, x1, u2f(s[2 * i]), u2f(s[2 * i + 1]), c, c, neg_m, neg_m);
        if ((i & 7) < S::kEmuPer8) {
          exp2_poly2(x0, x1, p0, p1);
        } else {
          p0 = ex2_approx(x0);
          p1 = ex2_approx(x1);
        }
        pk[i] = Elem<E>::pack2(p0, p1);
        Elem<E>::acc2(acc[2 * (i & 1)], acc[2 * (i & 1) + 1], pk[i]);
        if (i == 31) tmem_st32(tS, pk);
      }
      if constexpr (S::kPairs == 48) tmem_st16(tS + 32, pk + 32);
      l += (acc[0] + acc[1]) + (acc[2] + acc[3]);
      // O rescale (rare), once PV(j-1) has landed: committed with S(j+1) when
      // that tile exists, else (j = n-1) as the item's first PV-only batch.
      if (__any_sync(0xffffffffu, need)) {
        const bool ok = (j + 1 < n) ? warp_wait(&ctl->s_full[wg][(j + 1) & 1], s_parity(j + 1), abort_flag, a.status,
                                                kSiteODone, a.timeout_ns)
                                    : warp_wait(&ctl->pv_prev[wg], (base_bits >> 3) & 1, abort_flag, a.status,
                                                kSiteODone, a.timeout_ns);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * h, o);
          tmem_wait_ld_regs<32>(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(u2f(o[i]) * factor);
          tmem_st32(tO + 32 * h, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->p_full[wg][b]);
    }

    // The next item's hand-off while PV(n-1) runs.
    if (!next_item<D>(a, ctl, k + 1, &nxt)) return;
    have_nxt = true;
    if (n > 0) {
      if (!warp_wait(&ctl->pv_last[wg], (base_bits >> 2) & 1, abort_flag, a.status, kSiteODone, a.timeout_ns)) return;
      tc_fence_after();
      base_bits ^= (((n + 1) >> 1) & 1) | (((n >> 1) & 1) << 1) | 4u | (n > 1 ? 8u : 0u);
    }
    const float inv_l = 1.0f / l;
    const bool empty = lim < 0;
#pragma unroll
    for (int h = 0; h < D / 32; ++h) {
      uint32_t o[32];
      __syncwarp();
      if (n > 0) {
        tmem_ld32(tO + 32 * h, o);
        tmem_wait_ld_regs<32>(o);
      }
      if (valid) {
        uint4* dst = reinterpret_cast<uint4*>(out + 32 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (!empty) {
            v.x = Elem<E>::pack2(u2f(o[8 * i + 0]) * inv_l, u2f(o[8 * i + 1]) * inv_l);
            v.y = Elem<E>::pack2(u2f(o[8 * i + 2]) * inv_l, u2f(o[8 * i + 3]) * inv_l);
            v.z = Elem<E>::pack2(u2f(o[8 * i + 4]) * inv_l, u2f(o[8 * i + 5]) * inv_l);
            v.w = Elem<E>::pack2(u2f(o[8 * i + 6]) * inv_l, u2f(o[8 * i + 7]) * inv_l);
          }
          dst[i] = v;
        }
      }
    }
  }
}

// Items are numbered sequence by sequence, key head by key head, and within
// one from its last tokens to its first (the longest causal rows first).
struct Decoder {
  uint32_t seq0 = 0;    // sequences before it are scanned
  uint64_t before = 0;  // items of them
};

// The whole producer warp decodes item number `id`; false: past the last one.
template <int D>
__device__ __forceinline__ bool decode_item(const Args& a, Decoder& d, uint32_t id, Item* it) {
  const uint32_t lane = threadIdx.x & 31;
  const int item_tokens = 2 * static_cast<int>(a.tile_tokens);
  if (id < d.before) d = Decoder{};
  for (; d.seq0 < a.n_seqs; d.seq0 += 32) {
    const uint32_t s = d.seq0 + lane;
    int q0 = 0, lq = 0, k0 = 0, lk = 0;
    if (s < a.n_seqs) {
      q0 = __ldg(a.cu_q + s);
      k0 = __ldg(a.cu_k + s);
      const int q1 = __ldg(a.cu_q + s + 1), k1 = __ldg(a.cu_k + s + 1);
      if (q0 < 0 || q1 < q0 || k0 < 0 || k1 < k0 || q1 > static_cast<int>(a.total_q) ||
          k1 > static_cast<int>(a.total_k)) {
        atomicCAS(a.status, 0, static_cast<int>(kSiteBadOffsets));
      } else {
        lq = q1 - q0;
        lk = k1 - k0;
      }
    }
    const uint32_t tiles = static_cast<uint32_t>((static_cast<int64_t>(lq) + item_tokens - 1) / item_tokens);
    uint64_t inc = static_cast<uint64_t>(tiles) * a.kv_heads;
    const uint64_t mine = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= static_cast<uint32_t>(o)) inc += up;
    }
    const uint64_t first = d.before + inc - mine;
    const uint32_t hit = __ballot_sync(0xffffffffu, id >= first && id < first + mine);
    if (!hit) {
      d.before += __shfl_sync(0xffffffffu, inc, 31);
      continue;
    }
    const int src = __ffs(hit) - 1;
    const uint32_t local = static_cast<uint32_t>(id - __shfl_sync(0xffffffffu, first, src));
    const uint32_t n = __shfl_sync(0xffffffffu, tiles, src);
    q0 = __shfl_sync(0xffffffffu, q0, src);
    lq = __shfl_sync(0xffffffffu, lq, src);
    k0 = __shfl_sync(0xffffffffu, k0, src);
    lk = __shfl_sync(0xffffffffu, lk, src);
    it->head = local / n;
    const int t0 = static_cast<int>(n - 1 - local % n) * item_tokens;
    it->q_row = q0 + t0;
    it->tokens = lq - t0;
    it->k_row = k0;
    it->n_keys = lk;
    it->lim = t0 + lk - lq;
    it->n = max(wg_tiles<D>(a, *it, 0), wg_tiles<D>(a, *it, 1));
    return true;
  }
  return false;
}

// The producer warp, converged: lane 0 issues.
template <int D>
__device__ void producer_role(const Args& a, const CUtensorMap* tm_q, const CUtensorMap* tm_k,
                              const CUtensorMap* tm_v, uint8_t* sQ, uint8_t* sK, uint8_t* sV, Ctrl<D>* ctl) {
  using S = Shape<D>;
  volatile int* abort_flag = &ctl->abort_flag;
  const bool lead = (threadIdx.x & 31) == 0;
  uint32_t q_issued[2] = {0, 0};
  uint32_t g = 0;     // K/V tiles issued so far
  uint32_t k = 0;     // items posted
  uint32_t asked = 0; // try_cancel requests
  bool ok = true;
  Decoder dec;
  uint32_t id = blockIdx.x;
  const uint32_t q_bytes = a.tile_tokens * a.group * 128 * S::kHalves;
  auto post = [&](const Item& it) {
    const uint32_t slot = k % kItemSlots;
    if (k >= kItemSlots && !warp_wait(&ctl->item_empty[slot], ((k / kItemSlots) - 1) & 1, abort_flag, a.status,
                                      kSiteItemEmpty, a.timeout_ns))
      return false;
    if (lead) {
      ctl->item[slot] = it;
      mbar_arrive(&ctl->item_full[slot]);  // release: visible to the readers' acquire
    }
    __syncwarp();
    ++k;
    return true;
  };
  while (true) {
    // Ask for the next pending block; the answer is read after this item's loads.
    if (lead) {
      mbar_arrive_expect_tx(&ctl->next_full, 16);
      asm volatile(
          "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
              smem_u32(&ctl->next)),
          "r"(smem_u32(&ctl->next_full))
          : "memory");
    }
    ++asked;
    Item it;
    if (decode_item<D>(a, dec, id, &it)) {
      if (!post(it)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int wg = 0; wg < 2; ++wg) {
        if (!ok || wg_tiles<D>(a, it, wg) == 0) continue;
        const uint32_t qi = q_issued[wg];
        const uint32_t qb = qi % S::kQBufs;
        if (qi >= S::kQBufs && !warp_wait(&ctl->q_empty[wg][qb], ((qi / S::kQBufs) - 1) & 1, abort_flag, a.status,
                                          kSiteQEmpty, a.timeout_ns)) {
          ok = false;
          continue;
        }
        if (lead) {
          mbar_arrive_expect_tx(&ctl->q_full[wg][qb], q_bytes);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            tma_load_4d(tm_q, &ctl->q_full[wg][qb], sQ + (wg * S::kQBufs + qb) * S::kQTileBytes + h * S::kQHalf,
                        64 * h, 0, static_cast<int>(it.head), it.q_row + wg * static_cast<int>(a.tile_tokens));
        }
        q_issued[wg] = qi + 1;
      }
      for (uint32_t j = 0; ok && j < it.n; ++j, ++g) {
        const uint32_t st = g % S::kStages;
        if (g >= S::kStages && !warp_wait(&ctl->kv_empty[st], ((g / S::kStages) - 1) & 1, abort_flag, a.status,
                                          kSiteKvEmpty, a.timeout_ns)) {
          ok = false;
          break;
        }
        if (lead) {
          const int key = it.k_row + static_cast<int>(j) * S::kBN;
          mbar_arrive_expect_tx(&ctl->kv_full[st], 2 * S::kKvTileBytes);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            tma_load_3d(tm_k, &ctl->kv_full[st], sK + st * S::kKvTileBytes + h * S::kKvHalf, 64 * h,
                        static_cast<int>(it.head), key);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            tma_load_3d(tm_v, &ctl->kv_full[st], sV + st * S::kKvTileBytes + h * S::kKvHalf, 64 * h,
                        static_cast<int>(it.head), key);
        }
      }
      if (!ok) break;
    }
    if (!warp_wait(&ctl->next_full, (asked - 1) & 1, abort_flag, a.status, kSiteNext, a.timeout_ns)) {
      ok = false;
      break;
    }
    uint32_t got, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}\n"
        : "=r"(got), "=r"(x)
        : "r"(smem_u32(&ctl->next))
        : "memory");
    __syncwarp();
    fence_proxy_async_smem();  // the answer is read before the next request overwrites it
    if (!got) break;
    id = x;
  }
  if (ok) post(Item{kNoItem, 0, 0, 0, 0, 0, 0});
  // Every copy and answer this warp asked for lands before the CTA can exit.
  mbar_wait_teardown(&ctl->next_full, (asked - 1) & 1, a.status, kSiteNext);
  for (uint32_t t = g > S::kStages ? g - S::kStages : 0; t < g; ++t)
    mbar_wait_teardown(&ctl->kv_full[t % S::kStages], (t / S::kStages) & 1, a.status, kSiteKvFull);
#pragma unroll
  for (int wg = 0; wg < 2; ++wg) {
    const uint32_t qi = q_issued[wg];
    for (uint32_t t = qi > S::kQBufs ? qi - S::kQBufs : 0; t < qi; ++t)
      mbar_wait_teardown(&ctl->q_full[wg][t % S::kQBufs], (t / S::kQBufs) & 1, a.status, kSiteQFull);
  }
  __syncwarp();
}

// One MMA warp per softmax warpgroup, converged; elect.sync issues.
template <typename E, int D>
__device__ void mma_role(const Args& a, int wg, uint8_t* sQ, uint8_t* sK, uint8_t* sV, Ctrl<D>* ctl, uint32_t tmem) {
  using S = Shape<D>;
  constexpr int kBN = S::kBN;
  volatile int* abort_flag = &ctl->abort_flag;
  constexpr bool kBf16 = Elem<E>::kBf16;
  constexpr uint32_t idesc_qk = idesc_f16(kBf16, kBM, kBN, false, false);
  constexpr uint32_t idesc_pv = idesc_f16(kBf16, kBM, D, false, true);
  // K=16 steps advance a K-major operand by 32 B inside the 128-byte column
  // block, then to the next block; a 16-key step of V advances by 2048 B, and
  // V's second block of 64 columns lies a leading-dimension stride on.
  const uint64_t q_desc0 = sdesc_sw128(smem_u32(sQ + wg * S::kQBufs * S::kQTileBytes), 16, 1024);
  const uint64_t k_desc = sdesc_sw128(smem_u32(sK), 16, 1024);
  const uint64_t v_desc = sdesc_sw128(smem_u32(sV), S::kKvHalf, 1024);
  constexpr uint64_t kKvTileStep = S::kKvTileBytes >> 4;
  constexpr uint64_t kQTileStep = S::kQTileBytes >> 4;
  const uint32_t o_tmem = tmem + S::col_o(wg);
  uint32_t p_base0 = 0, p_base1 = 0;  // p_full completions before this item, per buffer
  uint32_t q_used = 0;
  RingPos<S::kStages> s_pos;   // next K/V tile to wait for (S products, or release)
  RingPos<S::kStages> pv_pos;  // next K/V tile whose V feeds a PV product
  bool ok = true;

  auto issue_s = [&](uint64_t q_desc, uint32_t st, int buf) {
    const uint64_t kd = k_desc + st * kKvTileStep;
    const uint32_t d = tmem + S::col_s(wg, buf);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
      umma_ss_elect(d, q_desc + (k >> 2) * (S::kQHalf >> 4) + 2 * (k & 3), kd + (k >> 2) * (S::kKvHalf >> 4) + 2 * (k & 3),
                    idesc_qk, k > 0 ? 1u : 0u);
  };
  auto issue_pv = [&](uint32_t st, int buf, bool acc) {
    const uint64_t vd = v_desc + st * kKvTileStep;
    const uint32_t p = tmem + S::col_s(wg, buf);
#pragma unroll
    for (int k = 0; k < kBN / 16; ++k)
      umma_ts_elect(o_tmem, p + 8 * k, vd + 128 * k, idesc_pv, (acc || k > 0) ? 1u : 0u);
  };
  auto kv_wait = [&](const RingPos<S::kStages>& r) {
    return warp_wait(&ctl->kv_full[r.stage], r.phase, abort_flag, a.status, kSiteKvFull, a.timeout_ns);
  };
  // Values behind the sequence's end become zero.  Both MMA warps write the
  // same zeros; a warp's own products are issued behind its fence.
  auto clear_tail = [&](uint32_t st, int keys) {
    uint8_t* v = sV + st * S::kKvTileBytes;
    const int lane = threadIdx.x & 31;
    for (int x = keys * 8 + lane; x < kBN * 8; x += 32) {
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h)
        *reinterpret_cast<uint4*>(v + h * S::kKvHalf + x * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
  };

  Item nxt{};
  bool have_nxt = false;
  auto fetch_next = [&](uint32_t k_next) {
    if (!have_nxt) {
      if (!next_item<D>(a, ctl, k_next, &nxt)) return false;
      have_nxt = true;
    }
    return true;
  };
  for (uint32_t k = 0; ok; ++k) {
    Item it;
    if (have_nxt) {
      it = nxt;
      have_nxt = false;
    } else if (!next_item<D>(a, ctl, k, &it)) {
      break;
    }
    if (it.q_row == kNoItem) break;
    const uint32_t n = wg_tiles<D>(a, it, wg);
    if (n > 0) {
      const uint32_t qb = q_used % S::kQBufs;
      if (!warp_wait(&ctl->q_full[wg][qb], (q_used / S::kQBufs) & 1, abort_flag, a.status, kSiteQFull, a.timeout_ns))
        break;
      tc_fence_after();
      const uint64_t q_desc = q_desc0 + qb * kQTileStep;
      // Keys of this warpgroup's last tile that belong to the sequence, if not all do.
      const int tail = it.n_keys - static_cast<int>(n - 1) * kBN;
      // S(0) and S(1) up front.  The commit after the item's last S also frees its Q buffer.
      for (uint32_t t = 0; t < 2 && t < n; ++t) {
        if (!kv_wait(s_pos)) {
          ok = false;
          break;
        }
        issue_s(q_desc, s_pos.stage, static_cast<int>(t));
        s_pos.next();
        umma_commit_elect(&ctl->s_full[wg][t]);
        if (t == n - 1) {
          umma_commit_elect(&ctl->q_empty[wg][qb]);
          if (!fetch_next(k + 1)) ok = false;
        }
      }
      for (uint32_t j = 0; ok && j < n; ++j) {
        const int b = static_cast<int>(j & 1);
        const uint32_t st = pv_pos.stage;  // V_j: waited on before S(j) was issued
        pv_pos.next();
        if (j + 1 == n && tail < kBN) clear_tail(st, tail);
        if (!warp_wait(&ctl->p_full[wg][b], ((b ? p_base1 : p_base0) + (j >> 1)) & 1, abort_flag, a.status,
                       kSitePFull, a.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        issue_pv(st, b, j > 0);
        if (j + 2 < n) {
          if (!kv_wait(s_pos)) {
            ok = false;
            break;
          }
          issue_s(q_desc, s_pos.stage, b);  // after PV(j) in this warp's order: P(j) is read first
          s_pos.next();
          umma_commit_elect(&ctl->s_full[wg][b]);
          if (j + 2 == n - 1) {
            umma_commit_elect(&ctl->q_empty[wg][qb]);
            if (!fetch_next(k + 1)) {
              ok = false;
              break;
            }
          }
        } else {
          umma_commit_elect(j + 1 == n ? &ctl->pv_last[wg] : &ctl->pv_prev[wg]);
        }
        umma_commit_elect(&ctl->kv_empty[st]);
      }
      p_base0 += (n + 1) >> 1;
      p_base1 += n >> 1;
      ++q_used;
    }
    // Tiles only the other warpgroup needs: released once they have landed.
    for (uint32_t j = n; ok && j < it.n; ++j, s_pos.next()) {
      if (!kv_wait(s_pos)) {
        ok = false;
        break;
      }
      mbar_arrive_elect(&ctl->kv_empty[s_pos.stage]);
    }
    pv_pos = s_pos;
  }
  // Every MMA this warp issued completes before TMEM is freed.
  umma_commit_elect(&ctl->drain[wg]);
  mbar_wait_teardown(&ctl->drain[wg], 0, a.status, kSiteODone);
  __syncwarp();
}

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 1)
    attn_varlen_sm100(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * S::kQBufs * S::kQTileBytes;
  uint8_t* sV = sK + S::kStages * S::kKvTileBytes;
  Ctrl<D>* ctl = reinterpret_cast<Ctrl<D>*>(sV + S::kStages * S::kKvTileBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&ctl->kv_full[s], 1);
      mbar_init(&ctl->kv_empty[s], 2);
    }
    for (int i = 0; i < 2; ++i) {
      for (int b = 0; b < S::kQBufs; ++b) {
        mbar_init(&ctl->q_full[i][b], 1);
        mbar_init(&ctl->q_empty[i][b], 1);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(&ctl->s_full[i][b], 1);
        mbar_init(&ctl->p_full[i][b], kBM / 32);
      }
      mbar_init(&ctl->pv_prev[i], 1);
      mbar_init(&ctl->pv_last[i], 1);
      mbar_init(&ctl->drain[i], 1);
    }
    for (int i = 0; i < kItemSlots; ++i) {
      mbar_init(&ctl->item_full[i], 1);
      mbar_init(&ctl->item_empty[i], kItemReaders);
    }
    mbar_init(&ctl->next_full, 1);
    ctl->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == kTmemWarp) {
    tmem_alloc(&ctl->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;

  if (warp < 8) {
    regs_inc<kSoftmaxRegs>();
    softmax_role<E, D>(a, ctl, tmem, warp, lane);
  } else {
    regs_dec<kControlRegs>();
    if (warp == kProducerWarp)
      producer_role<D>(a, &tm_q, &tm_k, &tm_v, sQ, sK, sV, ctl);
    else if (warp == kMmaWarp0 || warp == kMmaWarp0 + 1)
      mma_role<E, D>(a, warp - kMmaWarp0, sQ, sK, sV, ctl, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kTmemWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

bool encode(CUtensorMap* map, bool bf16, const void* base, uint32_t rank, const cuuint64_t* dims,
            const cuuint64_t* strides, const cuuint32_t* box, std::string* err) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) {
    if (err) *err = "cuTensorMapEncodeTiled unavailable";
    return false;
  }
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS && err) *err = "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r));
  return r == CUDA_SUCCESS;
}

template <typename E, int D>
cudaError_t launch(cudaStream_t stream, const VarlenIO& io, const Args& a, uint32_t grid, std::string* err) {
  using S = Shape<D>;
  CUtensorMap mq, mk, mv;
  // Queries as (D, heads of a group, key heads, tokens); keys and values as (D, key heads, tokens).
  const cuuint64_t qd[4] = {D, a.group, a.kv_heads, a.total_q};
  const cuuint64_t qs[3] = {D * 2, static_cast<cuuint64_t>(a.group) * D * 2, io.q_stride * 2};
  const cuuint32_t qb[4] = {64, a.group, 1, a.tile_tokens};
  const cuuint64_t kd[3] = {D, a.kv_heads, a.total_k ? a.total_k : 1};  // no keys at all: a map that nothing loads from
  const cuuint64_t ks[2] = {D * 2, io.k_stride * 2}, vs[2] = {D * 2, io.v_stride * 2};
  const cuuint32_t kb[3] = {64, 1, S::kBN};
  if (!encode(&mq, Elem<E>::kBf16, io.q, 4, qd, qs, qb, err) || !encode(&mk, Elem<E>::kBf16, io.k, 3, kd, ks, kb, err) ||
      !encode(&mv, Elem<E>::kBf16, io.v, 3, kd, vs, kb, err))
    return cudaErrorInvalidValue;
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(attn_varlen_sm100<E, D>),
                                            static_cast<int>(smem_bytes<D>()));
  if (e != cudaSuccess) return e;
  attn_varlen_sm100<E, D><<<grid, kThreads, smem_bytes<D>(), stream>>>(mq, mk, mv, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention_varlen(cudaStream_t stream, int code, uint32_t d, const VarlenIO& io, float scale,
                                    int* status, uint64_t timeout_ns, std::string* err) {
  Args a{};
  a.out = io.out;
  a.cu_q = io.cu_q;
  a.cu_k = io.cu_k;
  a.n_seqs = io.n_seqs;
  a.total_q = io.total_q;
  a.total_k = io.total_k;
  a.group = io.q_heads / io.kv_heads;
  a.kv_heads = io.kv_heads;
  a.tile_tokens = kBM / a.group;
  a.causal = io.causal;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status;
  a.timeout_ns = timeout_ns;
  // Every item the offsets can make: ceil(Lq / item) per sequence, summed.
  const uint64_t items =
      (static_cast<uint64_t>(io.total_q) / (2 * a.tile_tokens) + std::min(io.n_seqs, io.total_q)) * io.kv_heads;
  if (items > 0x7fffffffull) {
    if (err) *err = "too many work items";
    return cudaErrorInvalidValue;
  }
  VarlenIO use = io;
  if (io.total_k == 0) {
    use.k = use.v = io.q;
    use.k_stride = use.v_stride = io.q_stride;
  }
  const uint32_t grid = static_cast<uint32_t>(items);
  if (code == kBF16)
    return d == 64 ? launch<__nv_bfloat16, 64>(stream, use, a, grid, err)
                   : launch<__nv_bfloat16, 128>(stream, use, a, grid, err);
  return d == 64 ? launch<__half, 64>(stream, use, a, grid, err) : launch<__half, 128>(stream, use, a, grid, err);
}

}  // namespace hs
