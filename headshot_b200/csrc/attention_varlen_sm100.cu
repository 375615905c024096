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
// - The grid covers every item the packed rows can hold; a scheduler warp takes
//   over the next pending block with clusterlaunchcontrol.try_cancel while the
//   CTA works on the current item.  Scheduling is dynamic without a counter in
//   memory, so launches share nothing, and costly items go out first.  Which
//   sequence an item belongs to is found from the offsets on the device.
// - Under a causal mask each warpgroup stops at its own last key tile; tiles
//   that cross the diagonal or the sequence's end are masked element by element.
// - The keys of a tile that lie behind the sequence belong to the next one:
//   their scores are masked, and their values, which the PV product would
//   still multiply by zero, are overwritten with zeros in shared memory, so
//   infinities or NaN there cannot reach the result.
//
// Head_dim 64: 96-key tiles; 128: 64-key tiles, since two f32 accumulators of
// 128 columns leave 256 of TMEM's 512 columns for the four score buffers.
// Rounding: P is rounded to the storage type for the PV product; statistics,
// the row sum (of the unrounded P, in packed adds: summing the rounded P costs
// 3 % of the speed at 128 and 3 % at 64) and accumulators are f32.
//
// What bounds it (8,192 tokens, 32/8 x 128, not causal, one burst at 1,965
// MHz: 852 to 874 us on two GPUs, 1,258 to 1,290 TFLOP/s): per pair of 128 x
// 64 tiles 1,910 cycles and more, of which the tensor core's share is 1,260
// (64-column score products run at two thirds of its rate) and the
// exponentials' on the MUFU 900.  No pipe is full (tensor 67 %, XU 58 %,
// issue 53 % of the active cycles): a softmax warp spends most of them in
// the exponentials (both warpgroups at the same time, so at half the MUFU's
// rate each), the rest in the maximum, in waits for scores and in the
// hand-over.  Under load the 1,000 W cap takes the clock to 1,510 MHz: 1,139
// TFLOP/s for a causal prompt of 16,384.  Head_dim 64: 817 to 834 TFLOP/s
// for 16,384 tokens, 16 x 64, not causal; on 8,192 causal tokens XU 55 %,
// issue 58 %, tensor 37 % of the active cycles, and 20 % of the time SMs
// wait for the last items.  12 images of 261 to 1,374 tokens: XU 43 %, issue
// 50 %, SMs active for 80 % of the time.  Keys are not split: few queries
// onto a long history load few SMs (16 onto 100,000 keys, 32/8 x 128: 8
// CTAs, 934 us; the keys' bytes take 63).  Every CTA looks the offsets
// through once for the longest run and then class by class, 32 sequences at
// a time, which grows with the sequences.  An item's start and end cost
// about 6,000 cycles, three 96-key tiles' worth, and the GPU hands out about
// 28 pending blocks a microsecond, which bounds thousands of items that are
// shorter than 5 us each.  (Dealing half to seven eighths of the items out
// by block index instead: 9 % faster there, up to 7 % slower on ragged
// prompts.)
// Steps kept, on these two in TFLOP/s: 1,215 / 790 -> tested waits 1,240 /
// 798 -> the next K/V tile awaited before P 1,278 / 825 -> P stored 16
// columns at a time 1,312 / 830 -> the FMA pipe's share last of each 16
// pairs, masked weights exactly zero 1,329 / 837 -> exponents of score
// differences, right for any finite score, 1,290 / 834 where the step before
// reached 1,333 / 850.  Built and not kept, against the 1,215 / 790:
//   head_dim 128 with 128-key tiles and one score buffer (1,079; with one MMA
//     warp for both warpgroups 1,170, without splitting P's hand-over 1,251 in
//     a burst, 1,052 against 1,141 at the power cap)
//   one MMA warp for both warpgroups, 64-key tiles (970 / 747)
//   the warpgroups' exponentials taking turns (1,175 / 720)
//   each tile's exponentials interleaved with the next one's maximum, three
//     64-key score buffers at head_dim 64 (806 / 748)
//   four MMAs per election (1,214 / 781 to 801)
#include <cuda.h>

#include <float.h>

#include <algorithm>

#include "hs_internal.h"
#include "hs_ptx.cuh"

namespace hs {
namespace {

constexpr int kBM = 128;  // query rows per tile / softmax warpgroup
constexpr int kItemReaders = 8 + 2 + 1;  // one arrival per softmax warp, per MMA warp and from the producer
constexpr int kThreads = 384;
constexpr uint32_t kLaunchRegs = 168;  // 65536 / 384 rounded down to a multiple of 8
constexpr uint32_t kSoftmaxRegs = 216;
constexpr uint32_t kControlRegs = 72;
static_assert(2 * kSoftmaxRegs + kControlRegs <= 3 * kLaunchRegs, "setmaxnreg split exceeds the launch budget");
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp0 = 9;
constexpr int kSchedWarp = 11;  // items; also the TMEM owner
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: p <= 2^8 between rescales

template <int D>
struct Shape {
  static constexpr int kBN = D == 64 ? 96 : 64;  // keys per tile: 4 kBN + 2 D columns of TMEM
  static constexpr int kPairs = kBN / 2;
  static constexpr int kSlots = D == 64 ? 6 : 5;  // K/V tiles in shared memory
  static constexpr int kQBufs = D == 64 ? 2 : 1;
  static constexpr int kHalves = D / 64;          // 128-byte column blocks of a row
  static constexpr int kQTileBytes = kBM * D * 2;
  static constexpr int kKvTileBytes = kBN * D * 2;
  static constexpr int kSlotBytes = 2 * kKvTileBytes;
  static constexpr uint32_t kQHalf = kBM * 128;   // bytes from one column block to the next
  static constexpr uint32_t kKvHalf = kBN * 128;
  // Of every 16 exponential pairs, the last this many run on the FMA pipe.
  // 8,192 tokens of 32/8 x 128 in a burst: 1 of 16 1,245, 2 1,329, 3 1,292
  // TFLOP/s; 16,384 of 16 x 64: 2 775, 4 837, 5 837, 6 822.  The same share
  // at the start of each 16 or each 8 loses 3 to 6 %.
  static constexpr int kEmuPer16 = D == 64 ? 4 : 2;
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

// One unit of work, as the scheduler decodes it.
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
  uint64_t kv_full[S::kSlots];
  uint64_t kv_empty[S::kSlots];
  uint64_t q_full[2][S::kQBufs];
  uint64_t q_empty[2][S::kQBufs];
  uint64_t s_full[2][2];
  uint64_t p_full[2][2];
  uint64_t pv_prev[2];
  uint64_t pv_last[2];
  uint64_t drain[2];
  uint64_t item_full;   // the next item is there
  uint64_t item_empty;  // every reader took it
  uint64_t next_full;
  uint4 next;  // try_cancel's answer
  Item item;
  uint32_t tmem_base;
  int abort_flag;
};

template <int D>
constexpr size_t smem_bytes() {
  using S = Shape<D>;
  return 1024 + 2 * S::kQBufs * S::kQTileBytes + S::kSlots * S::kSlotBytes + sizeof(Ctrl<D>);
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
  int out_sectors;  // out is 32-byte aligned
  float scale_log2;
  int* status;
  uint64_t timeout_ns;
};

__device__ __forceinline__ float u2f(uint32_t u) { return __uint_as_float(u); }

template <int kSlots>
struct RingPos {
  uint32_t slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  }
};

// Bounded wait whose outcome is the same for all 32 lanes.  Tests first: a
// phase that is complete, the common case, costs one test and a vote (+2 %).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status,
                                          int site, uint64_t timeout_ns) {
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
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

// Item k for a reader warp (all lanes).
template <int D>
__device__ __forceinline__ bool next_item(const Args& a, Ctrl<D>* ctl, uint32_t k, Item* item) {
  if (!warp_wait(&ctl->item_full, k & 1, &ctl->abort_flag, a.status, kSiteItemFull, a.timeout_ns)) return false;
  const volatile Item* src = &ctl->item;
  item->q_row = src->q_row;
  item->tokens = src->tokens;
  item->k_row = src->k_row;
  item->n_keys = src->n_keys;
  item->lim = src->lim;
  item->head = src->head;
  item->n = src->n;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&ctl->item_empty);
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

// The largest of three; NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair on the FMA pipe: the same reduction and cubic as
// attn_fwd_sm100's (max relative error 8.3e-5).  Below 2^-127 the exponent sum
// turns negative and the result is 0, as the MUFU's is below 2^-126 (add and
// maximum are one instruction): a masked weight has to be 0 and not merely
// tiny, since a bf16 value reaches 2^128.
constexpr float kExpMagic = 12582912.0f;  // 1.5 * 2^23
constexpr float kExpC0 = 0.99991959f;
constexpr float kExpC1 = 0.69326216f;
constexpr float kExpC2 = 0.24271429f;
constexpr float kExpC3 = 0.05521307f;

__device__ __forceinline__ void exp2_poly2(float x0, float x1, float& y0, float& y1) {
  x0 = fmaxf(x0, -150.f);
  x1 = fmaxf(x1, -150.f);
  float t0, t1, r0, r1, f0, f1, p0, p1;
  add2(t0, t1, x0, x1, kExpMagic, kExpMagic);
  add2(r0, r1, t0, t1, -kExpMagic, -kExpMagic);
  fma2(f0, f1, r0, r1, -1.f, -1.f, x0, x1);
  fma2(p0, p1, f0, f1, kExpC3, kExpC3, kExpC2, kExpC2);
  fma2(p0, p1, p0, p1, f0, f1, kExpC1, kExpC1);
  fma2(p0, p1, p0, p1, f0, f1, kExpC0, kExpC0);
  y0 = __int_as_float(__viaddmax_s32(__float_as_int(p0), __float_as_int(t0) << 23, 0));
  y1 = __int_as_float(__viaddmax_s32(__float_as_int(p1), __float_as_int(t1) << 23, 0));
}

__device__ __forceinline__ void store32(void* dst, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
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
  const float threshold = fminf(kRescaleThreshold / c, 1e30f);  // of scores before the scale
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
      bool need = false;
      float m4[4] = {u2f(s[0]), u2f(s[1]), u2f(s[2]), u2f(s[3])};
#pragma unroll
      for (int i = 4; i < kBN; i += 2) m4[(i >> 1) & 3] = max3_nan(m4[(i >> 1) & 3], u2f(s[i]), u2f(s[i + 1]));
      const float m_tile = max3_nan(max3_nan(m4[0], m4[0], m4[1]), m4[2], m4[3]);
      const float m_old = m_run;
      if (j == 0 || m_tile > m_run + threshold) {
        m_run = m_tile;
        need = j > 0;
      }
      // A row that sees no key has m_run = -inf and turns into NaN here: its
      // output is set to zero below, and no other row reads it.
      // The exponents are (s - m) c, right for any finite score.  (s c - m c in one
      // fused step is 1.3 to 2.6 % faster on long prompts, but m c rounds away
      // binades from 2^26 on; telling such rows apart costs more than the second
      // step: 16 % by a branch here, 5 % by a flag that only reports them.)
      const float neg_m = -m_run;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t pk[S::kPairs];
#pragma unroll
      for (int i = 0; i < S::kPairs; ++i) {
        float x0, x1, p0, p1;
        add2(x0, x1, u2f(s[2 * i]), u2f(s[2 * i + 1]), neg_m, neg_m);
        mul2(x0, x1, x0, x1, c, c);
        if ((i & 15) >= 16 - S::kEmuPer16) {
          exp2_poly2(x0, x1, p0, p1);
        } else {
          p0 = ex2_approx(x0);
          p1 = ex2_approx(x1);
        }
        pk[i] = Elem<E>::pack2(p0, p1);
        add2(acc[2 * (i & 1)], acc[2 * (i & 1) + 1], acc[2 * (i & 1)], acc[2 * (i & 1) + 1], p0, p1);
        if (i % 16 == 15) tmem_st16(tS + i - 15, pk + i - 15);
      }
      float sum = (acc[0] + acc[1]) + (acc[2] + acc[3]);
      // A NaN score (or one past f32) makes the row's sum, and so its output, NaN
      // through its maximum: the FMA pipe's exponential alone would clamp it to a
      // weight of zero, and the key would be gone without a trace.
      sum = fmaf(max3_nan(m_tile, m_tile, -FLT_MAX), 0.f, sum);
      // O rescale (rare), once PV(j-1) has landed: committed with S(j+1) when
      // that tile exists, else (j = n-1) as the item's first PV-only batch.
      if (__any_sync(0xffffffffu, need)) {
        const bool ok = (j + 1 < n) ? warp_wait(&ctl->s_full[wg][(j + 1) & 1], s_parity(j + 1), abort_flag, a.status,
                                                kSiteODone, a.timeout_ns)
                                    : warp_wait(&ctl->pv_prev[wg], (base_bits >> 3) & 1, abort_flag, a.status,
                                                kSiteODone, a.timeout_ns);
        if (!ok) {
          tmem_wait_st();  // P's stores land before TMEM is freed
          return;
        }
        tc_fence_after();
        const float factor = need ? ex2_approx((m_old - m_run) * c) : 1.f;
        l *= factor;
#pragma unroll
        for (int h = 0; h < D / 16; ++h) {
          uint32_t o[16];
          tmem_ld16(tO + 16 * h, o);
          tmem_wait_ld_regs<16>(o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(u2f(o[i]) * factor);
          tmem_st16(tO + 16 * h, o);
        }
      }
      l += sum;
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
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = empty ? 0u : Elem<E>::pack2(u2f(o[2 * i]) * inv_l, u2f(o[2 * i + 1]) * inv_l);
        // The lanes' rows lie apart, so a store's cost is the sectors it touches:
        // whole 32-byte ones where the base allows (400 sequences of 256 tokens,
        // 16 x 64: 284 -> 262 us).
        if (a.out_sectors) {
          store32(out + 32 * h, w);
          store32(out + 32 * h + 16, w + 8);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            reinterpret_cast<uint4*>(out + 32 * h)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      }
    }
  }
}

// Items are numbered from costly to cheap, so that the last ones to start are
// short: by classes of their key count (64 << c, each twice the next), within
// a class sequence by sequence, last tokens first, and the key heads of the
// same tokens side by side (one causal prompt of 4,096 tokens, 32/8 x 128, in
// sequence order head by head: a third of the SM time idle).
struct Decoder {
  int cls = 0;          // classes above it are done
  uint32_t seq0 = 0;    // and in it the sequences before seq0,
  uint32_t before = 0;  // with this many items in all
};

// Lengths of sequence s, zero if its offsets are out of order or range.
__device__ __forceinline__ void seq_of(const Args& a, uint32_t s, int* q0, int* lq, int* k0, int* lk) {
  *q0 = *lq = *k0 = *lk = 0;
  if (s >= a.n_seqs) return;
  const int q = __ldg(a.cu_q + s), q1 = __ldg(a.cu_q + s + 1), k = __ldg(a.cu_k + s), k1 = __ldg(a.cu_k + s + 1);
  if (q < 0 || q1 < q || k < 0 || k1 < k || q1 > static_cast<int>(a.total_q) || k1 > static_cast<int>(a.total_k)) {
    atomicCAS(a.status, 0, static_cast<int>(kSiteBadOffsets));
    return;
  }
  *q0 = q;
  *lq = q1 - q;
  *k0 = k;
  *lk = k1 - k;
}

// Items of a sequence (of n) with at most `keys` keys: its first ones.
__device__ __forceinline__ int items_within(const Args& a, int n, int lq, int lk, int keys, int item_tokens) {
  if (lk <= keys) return n;
  if (!a.causal) return 0;
  return max(0, (keys - (lk - lq)) / item_tokens);
}

// Whole warp.  Decodes item number `id`; false: past the last one.
template <int D>
__device__ __forceinline__ bool decode_item(const Args& a, Decoder& d, uint32_t id, Item* it) {
  const uint32_t lane = threadIdx.x & 31;
  const int item_tokens = 2 * static_cast<int>(a.tile_tokens);
  for (; d.cls >= 0; --d.cls, d.seq0 = 0) {
    for (; d.seq0 < a.n_seqs; d.seq0 += 32) {
      int q0, lq, k0, lk;
      seq_of(a, d.seq0 + lane, &q0, &lq, &k0, &lk);
      const int n = static_cast<int>((static_cast<uint32_t>(lq) + item_tokens - 1) / item_tokens);
      const int high = items_within(a, n, lq, lk, d.cls >= 25 ? 0x7fffffff : 64 << d.cls, item_tokens);
      const int low = d.cls > 0 ? items_within(a, n, lq, lk, 32 << d.cls, item_tokens) : 0;
      const uint32_t mine = static_cast<uint32_t>(high - low) * a.kv_heads;
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= static_cast<uint32_t>(o)) inc += up;
      }
      const uint32_t local = id - (d.before + inc - mine);
      const uint32_t hit = __ballot_sync(0xffffffffu, local < mine);
      if (!hit) {
        d.before += __shfl_sync(0xffffffffu, inc, 31);
        continue;
      }
      const int src = __ffs(hit) - 1;
      const int t0 = (high - 1 - static_cast<int>(local / a.kv_heads)) * item_tokens;
      it->head = __shfl_sync(0xffffffffu, local % a.kv_heads, src);
      it->q_row = __shfl_sync(0xffffffffu, q0 + t0, src);
      it->tokens = __shfl_sync(0xffffffffu, lq - t0, src);
      it->k_row = __shfl_sync(0xffffffffu, k0, src);
      it->n_keys = __shfl_sync(0xffffffffu, lk, src);
      it->lim = __shfl_sync(0xffffffffu, t0 + lk - lq, src);
      it->n = max(wg_tiles<D>(a, *it, 0), wg_tiles<D>(a, *it, 1));
      return true;
    }
  }
  return false;
}

// The scheduler warp, converged: decodes this block's item, then the items of
// the pending blocks it takes over, one ahead of the readers.
template <int D>
__device__ void scheduler_role(const Args& a, Ctrl<D>* ctl) {
  volatile int* abort_flag = &ctl->abort_flag;
  const bool lead = (threadIdx.x & 31) == 0;
  uint32_t k = 0;      // items posted
  uint32_t asked = 0;  // try_cancel requests
  // The class of the longest key run.
  int most = 0;
  for (uint32_t s = threadIdx.x & 31; s < a.n_seqs; s += 32) {
    int q0, lq, k0, lk;
    seq_of(a, s, &q0, &lq, &k0, &lk);
    most = max(most, lk);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  const int top = most > 64 ? 26 - __clz(most - 1) : 0;  // smallest c with most <= 64 << c
  Decoder dec{top, 0, 0};
  auto post = [&](const Item& it) {
    if (k > 0 &&
        !warp_wait(&ctl->item_empty, (k - 1) & 1, abort_flag, a.status, kSiteItemEmpty, a.timeout_ns))
      return false;
    if (lead) {
      ctl->item = it;
      mbar_arrive(&ctl->item_full);  // release: visible to the readers' acquire
    }
    __syncwarp();
    ++k;
    return true;
  };
  uint32_t id = blockIdx.x, last = 0;
  bool ok = true;
  while (true) {
    if (id < last) dec = Decoder{top, 0, 0};
    last = id;
    Item it;
    if (decode_item<D>(a, dec, id, &it) && !post(it)) {
      ok = false;
      break;
    }
    if (lead) {
      mbar_arrive_expect_tx(&ctl->next_full, 16);
      asm volatile(
          "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
              smem_u32(&ctl->next)),
          "r"(smem_u32(&ctl->next_full))
          : "memory");
    }
    ++asked;
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
  // The answer to every request lands before the CTA can exit.
  if (asked) mbar_wait_teardown(&ctl->next_full, (asked - 1) & 1, a.status, kSiteNext);
  __syncwarp();
}

// The producer warp, converged: lane 0 issues.
template <int D>
__device__ void producer_role(const Args& a, const CUtensorMap* tm_q, const CUtensorMap* tm_k,
                              const CUtensorMap* tm_v, uint8_t* sQ, uint8_t* sKv, Ctrl<D>* ctl) {
  using S = Shape<D>;
  volatile int* abort_flag = &ctl->abort_flag;
  const bool lead = (threadIdx.x & 31) == 0;
  uint32_t q_issued[2] = {0, 0};
  uint32_t g = 0;  // ring slots filled so far
  bool ok = true;
  const uint32_t q_bytes = a.tile_tokens * a.group * 128 * S::kHalves;
  for (uint32_t k = 0; ok; ++k) {
    Item it;
    if (!next_item<D>(a, ctl, k, &it) || it.q_row == kNoItem) break;
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
    for (uint32_t j = 0; ok && j < it.n; ++j) {
      const int key = it.k_row + static_cast<int>(j) * S::kBN;
      const uint32_t st = g % S::kSlots;
      if (g >= S::kSlots && !warp_wait(&ctl->kv_empty[st], ((g / S::kSlots) - 1) & 1, abort_flag, a.status,
                                       kSiteKvEmpty, a.timeout_ns)) {
        ok = false;
        break;
      }
      if (lead) {
        uint8_t* slot = sKv + st * S::kSlotBytes;
        mbar_arrive_expect_tx(&ctl->kv_full[st], S::kSlotBytes);
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
          tma_load_3d(tm_k, &ctl->kv_full[st], slot + h * S::kKvHalf, 64 * h, static_cast<int>(it.head), key);
          tma_load_3d(tm_v, &ctl->kv_full[st], slot + S::kKvTileBytes + h * S::kKvHalf, 64 * h,
                      static_cast<int>(it.head), key);
        }
      }
      ++g;
    }
  }
  // Every copy this warp asked for lands before the CTA can exit.
  for (uint32_t t = g > S::kSlots ? g - S::kSlots : 0; t < g; ++t)
    mbar_wait_teardown(&ctl->kv_full[t % S::kSlots], (t / S::kSlots) & 1, a.status, kSiteKvFull);
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
__device__ void mma_role(const Args& a, int wg, uint8_t* sQ, uint8_t* sKv, Ctrl<D>* ctl, uint32_t tmem) {
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
  const uint64_t k_desc = sdesc_sw128(smem_u32(sKv), 16, 1024);
  const uint64_t v_desc = sdesc_sw128(smem_u32(sKv) + S::kKvTileBytes, S::kKvHalf, 1024);
  constexpr uint64_t kSlotStep = S::kSlotBytes >> 4;
  constexpr uint64_t kQTileStep = S::kQTileBytes >> 4;
  const uint32_t o_tmem = tmem + S::col_o(wg);
  uint32_t p_base0 = 0, p_base1 = 0;  // p_full completions before this item, per buffer
  uint32_t q_used = 0;
  RingPos<S::kSlots> s_pos;   // next slot to wait for (score products, or release)
  RingPos<S::kSlots> pv_pos;  // next slot whose V feeds a PV product
  bool ok = true;

  auto issue_s = [&](uint64_t q_desc, uint32_t st, int buf) {
    const uint64_t kd = k_desc + st * kSlotStep;
    const uint32_t d = tmem + S::col_s(wg, buf);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
      umma_ss_elect(d, q_desc + (k >> 2) * (S::kQHalf >> 4) + 2 * (k & 3), kd + (k >> 2) * (S::kKvHalf >> 4) + 2 * (k & 3),
                    idesc_qk, k > 0 ? 1u : 0u);
  };
  auto issue_pv = [&](uint32_t st, int buf, bool acc) {
    const uint64_t vd = v_desc + st * kSlotStep;
    const uint32_t p = tmem + S::col_s(wg, buf);
#pragma unroll
    for (int k = 0; k < kBN / 16; ++k)
      umma_ts_elect(o_tmem, p + 8 * k, vd + 128 * k, idesc_pv, (acc || k > 0) ? 1u : 0u);
  };
  auto kv_wait = [&](const RingPos<S::kSlots>& r) {
    return warp_wait(&ctl->kv_full[r.slot], r.phase, abort_flag, a.status, kSiteKvFull, a.timeout_ns);
  };
  // Values behind the sequence's end become zero.  Both MMA warps write the
  // same zeros; a warp's own products are issued behind its fence.
  auto clear_tail = [&](uint32_t st, int keys) {
    uint8_t* v = sKv + st * S::kSlotBytes + S::kKvTileBytes;
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
        issue_s(q_desc, s_pos.slot, static_cast<int>(t));
        s_pos.next();
        umma_commit_elect(&ctl->s_full[wg][t]);
        if (t == n - 1) {
          umma_commit_elect(&ctl->q_empty[wg][qb]);
          if (!fetch_next(k + 1)) ok = false;
        }
      }
      for (uint32_t j = 0; ok && j < n; ++j) {
        const int b = static_cast<int>(j & 1);
        const uint32_t st = pv_pos.slot;  // V_j: waited on before S(j) was issued
        pv_pos.next();
        if (j + 1 == n && tail < kBN) clear_tail(st, tail);
        // The next score product's tile, waited for while P(j) is still being made.
        if (j + 2 < n && !kv_wait(s_pos)) {
          ok = false;
          break;
        }
        if (!warp_wait(&ctl->p_full[wg][b], ((b ? p_base1 : p_base0) + (j >> 1)) & 1, abort_flag, a.status,
                       kSitePFull, a.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        issue_pv(st, b, j > 0);
        if (j + 2 < n) {
          issue_s(q_desc, s_pos.slot, b);  // after PV(j) in this warp's order: P(j) is read first
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
      mbar_arrive_elect(&ctl->kv_empty[s_pos.slot]);
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
  uint8_t* sKv = sQ + 2 * S::kQBufs * S::kQTileBytes;
  Ctrl<D>* ctl = reinterpret_cast<Ctrl<D>*>(sKv + S::kSlots * S::kSlotBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kSlots; ++s) {
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
    mbar_init(&ctl->item_full, 1);
    mbar_init(&ctl->item_empty, kItemReaders);
    mbar_init(&ctl->next_full, 1);
    ctl->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == kSchedWarp) {
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
      producer_role<D>(a, &tm_q, &tm_k, &tm_v, sQ, sKv, ctl);
    else if (warp == kMmaWarp0 || warp == kMmaWarp0 + 1)
      mma_role<E, D>(a, warp - kMmaWarp0, sQ, sKv, ctl, tmem);
    else
      scheduler_role<D>(a, ctl);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kSchedWarp) {
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
  a.out_sectors = (reinterpret_cast<uintptr_t>(io.out) & 31u) == 0;
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
