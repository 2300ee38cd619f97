// Causal attention of packed sequences with grouped query heads (prompts, prompt chunks over a
// history, single tokens over a history), dense keys and values.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j),  j <= t + k_len - q_len
//
// One CTA takes one work item: one KV head, one or two tiles of 128 query rows, a range of keys.  A
// tile's rows are 128 / G tokens times the G query heads of the KV head, so the group's heads read
// each key tile once and a single token fills G rows.  The two softmax warpgroups work on each other's turn:
// the tensor cores make the scores of one while the weights of the other are made.
//   Two query tiles: one per warpgroup, four products per key tile, which is read once for both.
//   One query tile (batches too small to fill the SMs with pairs): the warpgroups take key tiles in turn, each
//   with its own reference, sum and accumulator, which are added at the end.  Four single tokens over 22K
//   keys: 30.6 us with one warpgroup, 27.9 us with both; 148 CTAs of 16 key tiles each: 65.2 and 48.6 us.
//
//   warps 0-3, 4-7   softmax, one row per thread; output of the rows
//   warp 8           issues the products
//   warp 9           loads tiles (TMA) into a ring of five or six 32 KB stages: K0 V0 K1 V1 ...
//   warps 10, 11     clean value tiles that some row does not see whole
//
// Bound, one 16K prompt of 32 + 8 heads (1.82 to 1.92 ms by the clock that the power limit leaves, about
// 1,150 to 1,200 TFLOP/s of the causal half's products): tensor cores and special-function units alike, neither
// hidden under the other.  128 keys for both tiles take about 3,170 cycles, of which the four products need 2,050 (8.4 M
// multiply-adds at 4,096 a cycle) and the exponentials 2,048 (32,768 at 16 a cycle); counters: 54% and 57%.  The rest
// is the latency of scores, weights and products after one another: a tile's weights are handed over whole.  Keys in
// units of 64 with two score buffers per tile took 4,500 (products with 64 columns wait for shared memory), two
// issuing warps and a share of the exponentials as polynomials on the FMA pipe were slower too.
// Bound, packed requests (12 of 1 to 2,500 tokens, 146 us): an item has 7 key tiles in the mean, and its
// start and end, about 7 us, stand beside 12 us of tiles.  CTAs that stay and take items in turn,
// with the next item's loads and first scores under the last one's end, gained that back for items of one or
// two key tiles only (9.1 instead of 9.9 us each) and lost a ring stage: 162 us where these took 155.
// Bound, single tokens: memory (100 MB; the floor is 15.3 us), launch, the first loads and the merge.
//
// Values that no row may see: keys past the item's range in its last tile belong to another
// sequence, and a masked weight of 0 times an infinity or NaN is NaN.  Such rows of the last tile are
// cleared before its product, and in tiles that some row sees only part of, rows with non-finite
// values that not every row sees are cleared and marked; rows that do see a marked key add it at the end.
//
// Long key ranges with few query rows are split into several items; their unnormalised rows are merged by
// merge_items_kernel.
#include <cuda_bf16.h>

#include <algorithm>
#include <exception>
#include <string>
#include <vector>

#include "tp_umma.cuh"

namespace tp {

constexpr int kKeys = 128;               // keys per tile
constexpr int kRing = 6;                 // K and V tiles in flight: six with one query tile, five with two
constexpr int kPartial = 3;              // partly visible tiles of one item at most: 127 + 255 keys
// Three warpgroups at 168 registers: 504 in all, of which the softmax threads, with a row of scores
// each, take 224 and the others 56.
constexpr int kPromptThreads = 384, kSoftmaxRegs = 224, kIssueRegs = 56;
constexpr int kPromptMl = kTileBytes + kRing * kTileBytes;  // byte offset of references and sums to exchange
constexpr int prompt_bars(bool pair) { return kPromptMl + (pair ? 0 : 2 * kTile * 8); }  // of the barriers
constexpr int prompt_smem(bool pair) { return prompt_bars(pair) + 512; }
constexpr int kRecordRows = 2 * kTile;   // rows of an item's partial record
// Tensor memory (a CTA holds all of it, so it starts at column 0): scores of tile t at 128 t.
constexpr uint32_t kScoreCol = 0, kOutCol = 256;

// One work item (eight words, made on the host and copied to the device).
struct PromptItem {
  int32_t q_row;     // first token in the packed queries
  int32_t q_tokens;  // tokens, at most two tiles' worth
  int32_t sees;      // keys of its sequence that the first token sees (may be <= 0); one more for each next
  int32_t k_row;     // the sequence's first key in the packed keys
  int32_t k_begin, k_end;  // this item's keys, relative to k_row
  int32_t slot;      // record of an item that is merged later, or -1
  int32_t pad;
};
// The records of one token block that was split: `n` of them from `slot`.
struct PromptMerge {
  int32_t q_row, q_tokens, slot, n;
};

struct PromptParams {
  CUtensorMap qmap, kmap, vmap;
  const PromptItem* items;
  const PromptMerge* merges;
  int hq, hkv, group, tile_tokens;
  int merged;                 // merge_items_kernel follows
  float scale_log2;
  const uint16_t *q, *k, *v;  // for listed keys
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  uint16_t* out;              // [tokens][hq][128]
  float* rec_o;               // [slot][hkv][32][256][4]: channel / 4, row
  float2* rec_ml;             // [slot][hkv][256]
  int* error;
};

template <bool kBf16>
__device__ __forceinline__ float widen(uint16_t u) {
  return kBf16 ? __uint_as_float(uint32_t(u) << 16) : __half2float(__ushort_as_half(u));
}
// Bit 15 or 31 is set where that 16-bit number of w has an exponent of all ones: one more carries into it.
template <bool kBf16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return kBf16 ? (w & 0x7f807f80u) + 0x00800080u : (w & 0x7c007c00u) + 0x04000400u;
}

// Rows [first, 128) of a value tile: clear those from `valid` (at most 128) on and those with a non-finite value,
// whose bits are set in `late`.  Two warps (`which` 0, 1) take pairs of rows in turn, 16 lanes to a row, with
// eight loads in flight.
template <bool kBf16>
__device__ void clean_values(uint8_t* tile, int first, int valid, int which, uint32_t* late) {
  const int lane = threadIdx.x & 31;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint8_t* at = tile + (lane >> 3 & 1) * kHalfTile + (lane & 7) * 16;  // this lane's chunk of row 0
  for (int r0 = first + 2 * which; r0 < kKeys; r0 += 32) {
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = r0 + 4 * i + (lane >> 4);
      x[i] = zero;
      if (row < valid) x[i] = *reinterpret_cast<const uint4*>(at + row * 128);
      else if (row < kKeys) *reinterpret_cast<uint4*>(at + row * 128) = zero;
    }
    uint32_t bad = 0;  // bit i: x[i] holds a non-finite value
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t any = not_finite<kBf16>(x[i].x) | not_finite<kBf16>(x[i].y) | not_finite<kBf16>(x[i].z) |
                           not_finite<kBf16>(x[i].w);
      if (any & 0x80008000u) bad |= 1u << i;
    }
    if (!__any_sync(0xffffffffu, bad)) continue;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t hits = __ballot_sync(0xffffffffu, bad >> i & 1) >> (lane & 16) & 0xffffu;  // of this lane's row
      if (hits) {
        const int row = r0 + 4 * i + (lane >> 4);
        *reinterpret_cast<uint4*>(at + row * 128) = zero;
        if ((lane & 15) == 0) atomicOr(late + (row >> 5), 1u << (row & 31));
      }
    }
  }
}

// kPair: items have up to two query tiles, one per softmax warpgroup.  Otherwise an item is one query
// tile whose key tiles the warpgroups take in turn, each with an accumulator.
template <bool kBf16, bool kPair>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_attention_kernel(const __grid_constant__ PromptParams P) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PromptItem it = P.items[blockIdx.x / P.hkv];
  const int kvh = blockIdx.x % P.hkv;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + prompt_bars(kPair));
  uint64_t *full = q_full + 1, *empty = full + kRing, *s_full = empty + kRing, *p_full = s_full + 2,
           *o_done = p_full + 2, *asked = o_done + 2, *clean = asked + kPartial, *met = clean + kPartial, *drained = met + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* stop = reinterpret_cast<int*>(tmem_slot + 1);
  uint32_t* late = tmem_slot + 2;  // [kPartial][4]: marked keys, from key partial * 128 on
  // The item for the end of the softmax threads, which have no registers for it while they work.
  volatile PromptItem* held = reinterpret_cast<PromptItem*>(late + 4 * kPartial);

  const int n_tiles = (it.k_end - it.k_begin + kKeys - 1) / kKeys;
  const int nt = kPair && it.q_tokens > P.tile_tokens ? 2 : 1;  // query tiles
  // With one query tile the second's memory belongs to the ring.
  constexpr int stages = kPair ? kRing - 1 : kRing;
  uint8_t* ring = smem + (kPair ? 2 : 1) * kTileBytes;
  // Tiles from `partial` on are not seen whole by every row (or end after the item's keys).
  const int whole = min(it.sees, it.k_end) - it.k_begin;
  const int partial = whole <= 0 ? 0 : whole / kKeys;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(o_done + i, 1);
    }
    for (int i = 0; i < kPartial; ++i) {
      mbar_init(asked + i, 1);
      mbar_init(clean + i, 2);
    }
    if (!kPair) mbar_init(met, 8);
    mbar_init(drained, 1);
    *stop = 0;
    held->q_row = it.q_row, held->q_tokens = it.q_tokens;
    held->k_row = it.k_row, held->k_begin = it.k_begin, held->slot = it.slot;
    for (int i = 0; i < 4 * kPartial; ++i) late[i] = 0;
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(tmem_slot, 512);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (tmem != 0 && threadIdx.x == 0) *stop = 1;  // all 512 columns: always at 0
  // merge_items_kernel waits for this grid itself; nothing else may start before it has completed.
  if (P.merged) asm volatile("griddepcontrol.launch_dependents;");

  if (warp < 8) {
    more_registers<kSoftmaxRegs>();
    const int t = warp >> 2;
    int r = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_addr = kScoreCol + 128 * t + lanes, o_addr = kOutCol + 128 * t + lanes;
    // Keys of the item that the row sees.  Rows that are not there see everything, so they ask for no masking;
    // they are not written.
    auto token = [&](int row) { return (kPair ? t * P.tile_tokens : 0) + row / P.group; };
    auto exists = [&](int row, int tok, int q_tokens) { return row < P.tile_tokens * P.group && tok < q_tokens; };
    const int limit = (exists(r, token(r), it.q_tokens) ? min(it.sees + token(r), it.k_end) : it.k_end) - it.k_begin;
    const bool live = __any_sync(0xffffffffu, exists(r, token(r), it.q_tokens));
    SoftmaxRow row;
    bool ok = true;
    int n = 0;  // tiles of this warpgroup so far: all of the item's, or every second one
    if constexpr (kPair) {  // two loops: one for both forms, with a variable step, cost pairs 2.5%
      if (t < nt) {
        for (int j = 0; j < n_tiles && ok; ++j) {
          ok = __all_sync(0xffffffffu, wait_bar(s_full + t, j & 1, stop));
          if (ok && live) {
            tmem_fence_after();
            ok = softmax_tile<kKeys, kBf16>(row, s_addr, o_addr, FirstN{limit - j * kKeys}, P.scale_log2, j == 0,
                                            [&] { return wait_bar(o_done + t, (j - 1) & 1, stop); });
            tmem_fence_before();
          }
          __syncwarp();
          if (ok && lane == 0) mbar_arrive(p_full + t);
        }
        n = n_tiles;
      }
    } else {
      for (int j = t; j < n_tiles && ok; j += 2, ++n) {
        ok = __all_sync(0xffffffffu, wait_bar(s_full + t, n & 1, stop));
        if (ok && live) {
          tmem_fence_after();
          ok = softmax_tile<kKeys, kBf16>(row, s_addr, o_addr, FirstN{limit - j * kKeys}, P.scale_log2, n == 0,
                                          [&] { return wait_bar(o_done + t, (n - 1) & 1, stop); });
          tmem_fence_before();
        }
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(p_full + t);
      }
    }
    if (ok && n) {
      ok = wait_bar(o_done + t, (n - 1) & 1, stop);
      for (int i = 0; i < n_tiles - partial; ++i) ok = ok && wait_bar(clean + i, 0, stop);
      ok = __all_sync(0xffffffffu, ok);
    }
    float2 other = make_float2(-INFINITY, 0.0f);
    if (!kPair && ok) {
      // Both warpgroups hold parts of the same rows: exchange references and sums, then each writes half
      // of the channels of both accumulators' weighted sum.
      float2* ml = reinterpret_cast<float2*>(smem + kPromptMl);
      ml[t * kTile + r] = make_float2(row.ref, row.sum);
      __syncwarp();
      if (lane == 0) mbar_arrive(met);
      ok = __all_sync(0xffffffffu, wait_bar(met, 0, stop));
      if (ok) other = ml[(t ^ 1) * kTile + r];
    }
    if (ok && live) {
      tmem_fence_after();
      const float top = kPair ? row.ref : fmaxf(row.ref, other.x);
      const float base = top == -INFINITY ? 0.0f : top;
      const float mine = kPair ? 1.0f : exp2_approx(row.ref - base), others = kPair ? 0.0f : exp2_approx(other.x - base);
      const float sum = kPair ? row.sum : mine * row.sum + others * other.y;
      const bool here = n > 0, there = !kPair && n_tiles > (t ^ 1);  // accumulators that hold something
      const bool marked = __any_sync(0xffffffffu, lane < 4 * kPartial && late[lane]);
      asm volatile("" : "+r"(r));  // computed again, not kept
      const int tok = token(r), head = kvh * P.group + r % P.group, slot = held->slot, k_begin = held->k_begin, k_row = held->k_row;
      const bool valid = exists(r, tok, held->q_tokens), merged = slot >= 0;
      const int64_t q_row = int64_t(held->q_row) + tok;
      const int64_t rec = int64_t(slot) * P.hkv + kvh;
      const int rec_row = (kPair ? t * kTile : 0) + r;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint8_t* dst = valid ? reinterpret_cast<uint8_t*>(P.out + (q_row * P.hq + head) * kD) : nullptr;
      // All of the row's channels at once (without pairs, this warpgroup's half of them): the loads and the
      // stages of shared memory wait for one another once, not every 32 channels (packed prompts 156 -> 153 us).
      constexpr int kC = kPair ? kD : kD / 2;
      const int c0 = kPair ? 0 : kC * t;
      float o[kC];
      if (here) {
#pragma unroll
        for (int c = 0; c < kC; c += 32) tmem_ld32(o_addr + c0 + c, o + c);
        tmem_wait_ld<kC>(o);
      } else {
#pragma unroll
        for (int i = 0; i < kC; ++i) o[i] = 0.0f;
      }
      if (!kPair) {
#pragma unroll
        for (int i = 0; i < kC; ++i) o[i] *= mine;
        if (there) {
          float x[kC];
#pragma unroll
          for (int c = 0; c < kC; c += 32) tmem_ld32(kOutCol + 128 * (t ^ 1) + lanes + c0 + c, x + c);
          tmem_wait_ld<kC>(x);
#pragma unroll
          for (int i = 0; i < kC; ++i) o[i] = fmaf(others, x[i], o[i]);
        }
      }
      if (marked && valid) {  // keys with non-finite values that this row sees
        for (int e = 0; e < kPartial * kKeys; ++e) {
          if (partial * kKeys + e >= limit) break;
          const int key = k_begin + partial * kKeys + e;
          if (!(late[e >> 5] >> (e & 31) & 1)) continue;
          const uint16_t* qr = P.q + q_row * P.q_t + head * P.q_h;
          const uint16_t* kr = P.k + (int64_t(k_row) + key) * P.k_t + kvh * P.k_h;
          const uint16_t* vr = P.v + (int64_t(k_row) + key) * P.v_t + kvh * P.v_h + c0;
          float dot = 0.0f;
          for (int d = 0; d < kD; ++d) dot = fmaf(widen<kBf16>(qr[d]), widen<kBf16>(kr[d]), dot);
          const float p = exp2_approx(fmaf(dot, P.scale_log2, -base));
#pragma unroll
          for (int i = 0; i < kC; ++i) o[i] = fmaf(p, widen<kBf16>(vr[i]), o[i]);
        }
      }
      __syncwarp();
      if (merged) {
        float4* to = reinterpret_cast<float4*>(P.rec_o) + (rec * 32 + c0 / 4) * kRecordRows + rec_row;
#pragma unroll
        for (int i = 0; i < kC / 4; ++i)
          if (valid) to[i * kRecordRows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else {
        // The query tile has been read: its memory carries the rows out, 64 bytes of 32 rows in each 2 KB.
        uint8_t* buf = smem + (kPair ? t * kTileBytes + (warp & 3) * (kTileBytes / 4) : warp * (kTileBytes / 8));
#pragma unroll
        for (int c = 0; c < kC; c += 8)
          *staged(buf + (c >> 5) * kStageRows, lane, c >> 3 & 3) =
              make_uint4(pack2<kBf16>(o[c] * inv, o[c + 1] * inv), pack2<kBf16>(o[c + 2] * inv, o[c + 3] * inv),
                         pack2<kBf16>(o[c + 4] * inv, o[c + 5] * inv), pack2<kBf16>(o[c + 6] * inv, o[c + 7] * inv));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = 8 * i + (lane >> 2);  // four lanes to a row
          uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), from));
          if (to) {
#pragma unroll
            for (int c = 0; c < kC; c += 32)
              *reinterpret_cast<uint4*>(to + 2 * (c0 + c) + 16 * (lane & 3)) = *staged(buf + (c >> 5) * kStageRows, from, lane & 3);
          }
        }
      }
      if (merged && valid && (kPair || t == 0)) P.rec_ml[rec * kRecordRows + rec_row] = make_float2(top, sum);
    }
    tmem_fence_before();
  } else if (fewer_registers<kIssueRegs>(); warp == 8) {
    if (n_tiles) {
      constexpr uint32_t kScores = mma_idesc(kBf16, kKeys, false), kOut = mma_idesc(kBf16, kD, true);
      const uint32_t q_lo = rows_lo(smem_u32(smem)), ring_addr = smem_u32(ring);
      auto scores = [&](int t, int q_tile, int stage) {  // one thread
        const uint32_t k_lo = rows_lo(ring_addr) + stage * (kTileBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * kHalfTile + (ks & 3) * 32) >> 4;
          mma_ss(kScoreCol + 128 * t, q_lo + q_tile * (kTileBytes >> 4) + off, k_lo + off, kScores, ks > 0);
        }
        mma_commit(s_full + t);
      };
      auto values = [&](int t, uint32_t v_lo, bool add) {  // one thread
#pragma unroll
        for (int ks = 0; ks < kKeys / 16; ++ks)
          mma_ts(kOutCol + 128 * t, kScoreCol + 128 * t + ks * 8, v_lo + ks * (2048 >> 4), kOut, add || ks > 0);
        mma_commit(o_done + t);
      };
      // Issuing blocks until the tensor cores take the product, so time spent waiting is time they idle:
      // key and value tiles are waited for one step ahead, in the gaps where the weights are not ready yet.
      bool ok = warp_wait(q_full, 0, stop);
      if constexpr (kPair) {
        int st = 0, ph = 0;  // stage and phase of the next tile in the ring
        auto next_tile = [&](bool cleaned, int j) {
          bool here = warp_wait(full + st, ph, stop);
          if (here && cleaned && j >= partial) here = warp_wait(clean + j - partial, 0, stop);
          st = st + 1 == stages ? (ph ^= 1, 0) : st + 1;
          return here;
        };
        ok = ok && next_tile(false, 0);
        if (ok) {
          tmem_fence_after();
          if (elect_one()) {
            for (int t = 0; t < nt; ++t) scores(t, t, 0);
            mma_commit(empty);
          }
          __syncwarp();
        }
        int sv = st;
        ok = ok && next_tile(true, 0);
        int sk = st;
        if (n_tiles > 1) ok = ok && next_tile(false, 1);
        for (int j = 0; j < n_tiles && ok; ++j) {
          const bool more = j + 1 < n_tiles;
          int sv_next = 0, sk_next = 0;
        const uint32_t v_lo = cols_lo(ring_addr, kHalfTile) + sv * (kTileBytes >> 4);
          for (int t = 0; t < nt && ok; ++t) {
            // The tile's weights times the values, then its next scores (over the weights: products
            // complete in order).
            ok = warp_wait(p_full + t, j & 1, stop);
            if (!ok) break;
            tmem_fence_after();
            if (elect_one()) {
              values(t, v_lo, j > 0);
              if (t == nt - 1) mma_commit(empty + sv);
              if (more) {
                scores(t, t, sk);
                if (t == nt - 1) mma_commit(empty + sk);
              }
            }
            __syncwarp();
            if (t == 0 && more) {
              sv_next = st;
              ok = next_tile(true, j + 1);
            }
          }
          if (ok && j + 2 < n_tiles) {
            sk_next = st;
            ok = next_tile(false, j + 2);
          }
          sv = sv_next;
          sk = sk_next;
        }
      } else {
        // Key tile j belongs to warpgroup j & 1, and its scores follow the values of tile j - 2.  No tile is
        // loaded into a stage before the one there has been used, so tiles may be waited for out of order.
        auto keys_here = [&](int j) { return j >= n_tiles || warp_wait(full + 2 * j % stages, 2 * j / stages & 1, stop); };
        auto values_here = [&](int j) {
          return j >= n_tiles || (warp_wait(full + (2 * j + 1) % stages, (2 * j + 1) / stages & 1, stop) &&
                                  (j < partial || warp_wait(clean + j - partial, 0, stop)));
        };
        for (int j = 0; j < min(2, n_tiles) && ok; ++j) {
          ok = keys_here(j);
          if (!ok) break;
          tmem_fence_after();
          if (elect_one()) {
            scores(j, 0, 2 * j);
            mma_commit(empty + 2 * j);
          }
          __syncwarp();
        }
        ok = ok && values_here(0) && keys_here(2);
        for (int j = 0; j < n_tiles && ok; ++j) {
          const int t = j & 1;
          ok = warp_wait(p_full + t, j >> 1 & 1, stop);
          if (!ok) break;
          tmem_fence_after();
          if (elect_one()) {
            const int sv = (2 * j + 1) % stages, sk = (2 * j + 4) % stages;
            values(t, cols_lo(ring_addr, kHalfTile) + sv * (kTileBytes >> 4), j > 1);
            mma_commit(empty + sv);
            if (j + 2 < n_tiles) {
              scores(t, 0, sk);
              mma_commit(empty + sk);
            }
          }
          __syncwarp();
          ok = values_here(j + 1) && keys_here(j + 3);
        }
      }
      if (elect_one()) mma_commit(drained);
      __syncwarp();
      drain_bar(drained, 0);
    }
    __syncwarp();
  } else if (warp == 9 && n_tiles) {
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, uint32_t(nt * P.tile_tokens * P.group * 256));
      for (int t = 0; t < nt; ++t)
        for (int h = 0; h < 2; ++h)
          tma_tile_3d(smem_u32(smem) + t * kTileBytes + h * kHalfTile, &P.qmap, h * 64, kvh * P.group,
                      it.q_row + t * P.tile_tokens, q_full);
    }
    int issued = 0;
    bool ok = true;
    for (int i = 0; i < 2 * n_tiles && ok; ++i) {
      const int stage = i % stages, use = i / stages;
      ok = use == 0 || warp_wait(empty + stage, (use - 1) & 1, stop);
      if (!ok) break;
      if (lane == 0) {
        const uint32_t dst = smem_u32(ring) + stage * kTileBytes;
        const CUtensorMap* map = i & 1 ? &P.vmap : &P.kmap;
        mbar_arrive_expect_tx(full + stage, kTileBytes);
        for (int h = 0; h < 2; ++h)
          tma_tile_3d(dst + h * kHalfTile, map, h * 64, kvh, it.k_row + it.k_begin + (i >> 1) * kKeys, full + stage);
        if ((i & 1) && (i >> 1) >= partial) mbar_arrive(asked + (i >> 1) - partial);
      }
      issued = i + 1;
    }
    // No copy may be in flight when the CTA ends.
    drain_bar(q_full, 0);
    for (int i = max(0, issued - stages); i < issued; ++i) drain_bar(full + i % stages, (i / stages) & 1);
  } else if (n_tiles) {
    for (int j = partial; j < n_tiles; ++j) {
      // The stage's barrier is at this tile's phase once the loader has asked for it.
      const int i = 2 * j + 1, stage = i % stages;
      if (!warp_wait(asked + j - partial, 0, stop) || !warp_wait(full + stage, (i / stages) & 1, stop)) break;
      const int key = j * kKeys, valid = min(kKeys, it.k_end - it.k_begin - key);
      clean_values<kBf16>(ring + stage * kTileBytes, min(valid, max(0, whole - key)), valid, warp - 10,
                          late + 4 * (j - partial));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(clean + j - partial);
    }
  }
  __syncthreads();
  if (warp == 8) {
    tmem_fence_after();
    tmem_free(tmem, 512);
  }
  if (threadIdx.x == 0 && *stop) *P.error = 1;
}

// Rows of split token blocks: 32 rows x 8 channels per block.
template <bool kBf16>
__global__ void __launch_bounds__(kMergeThreads, 4) merge_items_kernel(const __grid_constant__ PromptParams P) {
  const PromptMerge m = P.merges[blockIdx.x / P.hkv];
  const int kvh = blockIdx.x % P.hkv;
  const int tile_rows = P.tile_tokens * P.group;
  const int r0 = blockIdx.y * 32, t = r0 >> 7;  // rows of the record: tile t, row r0 & 127
  const int rows = min(min(32, tile_rows - (r0 & 127)), m.q_tokens * P.group - t * tile_rows - (r0 & 127));
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (rows <= 0) return;
  const int64_t rec = int64_t(m.slot) * P.hkv + kvh;
  MergePart p;
  if (!merge_records<false>(p, P.rec_ml + rec * kRecordRows + r0,
                            reinterpret_cast<const float4*>(P.rec_o) + (rec * 32 + 2 * blockIdx.z) * kRecordRows + r0,
                            int64_t(P.hkv) * kRecordRows, int64_t(P.hkv) * 32 * kRecordRows, kRecordRows, m.n, rows) ||
      int(threadIdx.x) >= rows)
    return;
  const int i = t * tile_rows + (r0 & 127) + threadIdx.x;
  const int64_t at = ((int64_t(m.q_row) + i / P.group) * P.hq + kvh * P.group + i % P.group) * kD + 8 * blockIdx.z;
  *reinterpret_cast<uint4*>(P.out + at) =
      make_uint4(pack2<kBf16>(p.acc[0], p.acc[1]), pack2<kBf16>(p.acc[2], p.acc[3]), pack2<kBf16>(p.acc[4], p.acc[5]),
                 pack2<kBf16>(p.acc[6], p.acc[7]));
}

// ----------------------------------------------------------------------------- host
static int tile_tokens_of(int group) { return kTile / group; }

// Tensor map of rows [tokens][heads][128] of 16-bit numbers, boxes of 64 channels.
static int rows_map(CUtensorMap* m, const void* p, int64_t tokens, int heads, int64_t t_stride, int64_t h_stride,
                    int box_heads, int box_tokens, bool bf16, const char* what) {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    else
      cudaGetLastError();
  });
  if (!enc) return fail(TP_ERR_CUDA, "tp_prompt_attention: the driver has no cuTensorMapEncodeTiled");
  // The stride of an axis of one entry is not used, but has to be a legal one.
  if (heads == 1) h_stride = kD;
  if (tokens == 1) t_stride = int64_t(heads) * kD;
  if (!p || uintptr_t(p) % 16 || t_stride % 8 || h_stride % 8 || t_stride < kD || h_stride < kD)
    return fail(TP_ERR_INVALID, std::string("tp_prompt_attention: ") + what +
                                    " rows must be contiguous and start on 16-byte boundaries");
  const cuuint64_t dims[3] = {cuuint64_t(kD), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides[2] = {cuuint64_t(h_stride * 2), cuuint64_t(t_stride * 2)};
  const cuuint32_t box[3] = {64, cuuint32_t(box_heads), cuuint32_t(box_tokens)};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TP_ERR_INVALID, std::string("tp_prompt_attention: cannot describe ") + what + " (CUresult " +
                                    std::to_string(int(r)) + ")");
  return TP_OK;
}

static size_t record_bytes(int64_t slots, int hkv) {
  return size_t(slots) * hkv * kRecordRows * (kD * sizeof(float) + sizeof(float2));
}

template <bool kBf16, bool kPair>
static int launch_prompt(const PromptParams& P, const tp_prompt_plan& plan, cudaStream_t s) {
  static bool allowed[64] = {};  // the attribute belongs to a device's copy of the kernel
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !allowed[dev])) {
    const int st = allow_kernel(reinterpret_cast<const void*>(prompt_attention_kernel<kBf16, kPair>), prompt_smem(kPair),
                                kPromptThreads, 2 * kSoftmaxRegs + kIssueRegs, "tp_prompt_attention");
    if (st != TP_OK) return st;
    if (dev < 64) allowed[dev] = true;
  }
  if (e != cudaSuccess) return fail(TP_ERR_CUDA, std::string("tp_prompt_attention: ") + cudaGetErrorString(e));
  if (plan.items)
    prompt_attention_kernel<kBf16, kPair><<<unsigned(plan.items) * plan.num_kv_heads, kPromptThreads, prompt_smem(kPair), s>>>(P);
  if (plan.merges) {
    const int rows = kPair ? kRecordRows : plan.block_tokens * P.group;
    e = launch_dependent(merge_items_kernel<kBf16>, dim3(unsigned(plan.merges) * plan.num_kv_heads, (rows + 31) / 32, kD / 8),
                         kMergeThreads, s, P);
    if (e != cudaSuccess) return fail(TP_ERR_CUDA, std::string("tp_prompt_attention: ") + cudaGetErrorString(e));
  }
  return check_launch("tp_prompt_attention");
}

static int make_plan(const int64_t* q_lens, const int64_t* k_lens, int32_t n_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                     tp_prompt_plan* plan, int32_t* words, size_t n_words) {
  if (!plan || n_seqs < 0 || (n_seqs && (!q_lens || !k_lens)))
    return fail(TP_ERR_INVALID, "tp_prompt_plan_make: NULL argument");
  if (num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads)
    return fail(TP_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads for GQA");
  const int group = num_q_heads / num_kv_heads;
  if (group > kTile) return fail(TP_ERR_UNSUPPORTED, "tp_prompt_plan_make: more than 128 query heads per KV head");
  int64_t tq = 0, tk = 0, pairs = 0;
  const int tile = tile_tokens_of(group);
  for (int i = 0; i < n_seqs; ++i) {
    if (q_lens[i] < 0 || k_lens[i] < 0) return fail(TP_ERR_INVALID, "tp_prompt_plan_make: negative length");
    tq += q_lens[i];
    tk += k_lens[i];
    if (tq > INT32_MAX / 2 || tk > INT32_MAX / 2)
      return fail(TP_ERR_INVALID, "tp_prompt_plan_make: more than 2^30 tokens");
    pairs += (q_lens[i] + 2 * tile - 1) / (2 * tile);
  }
  const int64_t sms = device_sms();
  // Two tiles per item, which halves the reads of each key tile, unless that leaves SMs idle.
  const int block = pairs * num_kv_heads >= sms ? 2 * tile : tile;
  struct Block {
    int32_t q_row, q_tokens, sees, k_row, k_end, tiles;
  };
  std::vector<Block> blocks;
  int64_t q_row = 0, k_row = 0, work = 0, longest = 0;
  for (int i = 0; i < n_seqs; ++i) {
    for (int64_t a = 0; a < q_lens[i]; a += block) {
      Block b;
      b.q_row = int32_t(q_row + a);
      b.q_tokens = int32_t(std::min<int64_t>(block, q_lens[i] - a));
      b.sees = int32_t(k_lens[i] - q_lens[i] + a + 1);
      b.k_row = int32_t(k_row);
      b.k_end = int32_t(std::max<int64_t>(0, int64_t(b.sees) + b.q_tokens - 1));  // at most k_lens[i]
      b.tiles = (b.k_end + kKeys - 1) / kKeys;
      work += b.tiles;
      longest = std::max<int64_t>(longest, b.tiles);
      blocks.push_back(b);
    }
    q_row += q_lens[i];
    k_row += k_lens[i];
  }
  // Key ranges: an item takes about `chunk` tiles.  Fewer blocks than SMs: as many items as fit one
  // wave, at least four tiles each (a record of 256 rows is written and read for each item).
  int64_t chunk = std::max<int64_t>(4, (work * num_kv_heads + sms - 1) / sms);
  auto parts_of = [&](int64_t tiles) { return 2 * tiles > 3 * chunk ? (tiles + chunk - 1) / chunk : int64_t(1); };
  if (int64_t(blocks.size()) * num_kv_heads < sms) {
    for (; chunk < longest; ++chunk) {
      int64_t n = 0;
      for (const Block& b : blocks) n += parts_of(b.tiles);
      if (n * num_kv_heads <= sms) break;
    }
  }
  std::vector<PromptItem> items;
  std::vector<PromptMerge> merges;
  int64_t slots = 0;
  for (const Block& b : blocks) {
    const int64_t parts = parts_of(b.tiles);
    const int64_t per = (b.tiles + parts - 1) / parts;
    int32_t n = 0;
    for (int64_t j = 0; j < std::max<int64_t>(1, b.tiles); j += std::max<int64_t>(1, per), ++n)
      items.push_back(PromptItem{b.q_row, b.q_tokens, b.sees, b.k_row, int32_t(j * kKeys),
                                 int32_t(std::min<int64_t>(b.k_end, (j + per) * kKeys)),
                                 parts > 1 ? int32_t(slots + n) : -1, 0});
    if (parts > 1) {
      merges.push_back(PromptMerge{b.q_row, b.q_tokens, int32_t(slots), n});
      slots += n;
    }
  }
  // Longest items first: the CTAs are started in this order, so short ones fill the end.
  std::stable_sort(items.begin(), items.end(), [](const PromptItem& a, const PromptItem& b) {
    return (a.k_end - a.k_begin + kKeys - 1) / kKeys > (b.k_end - b.k_begin + kKeys - 1) / kKeys;
  });
  if (int64_t(items.size()) * num_kv_heads > INT32_MAX || slots > INT32_MAX / 2)
    return fail(TP_ERR_UNSUPPORTED, "tp_prompt_plan_make: too many work items");
  plan->num_q_heads = num_q_heads;
  plan->num_kv_heads = num_kv_heads;
  plan->q_tokens = tq;
  plan->k_tokens = tk;
  plan->items = int32_t(items.size());
  plan->merges = int32_t(merges.size());
  plan->block_tokens = block;
  plan->words = items.size() * (sizeof(PromptItem) / 4) + merges.size() * (sizeof(PromptMerge) / 4);
  plan->workspace_bytes = 256 + record_bytes(slots, num_kv_heads);
  if (!words) return TP_OK;
  if (n_words < plan->words) return fail(TP_ERR_INVALID, "tp_prompt_plan_make: the word buffer is too small");
  std::copy_n(reinterpret_cast<const int32_t*>(items.data()), items.size() * (sizeof(PromptItem) / 4), words);
  std::copy_n(reinterpret_cast<const int32_t*>(merges.data()), merges.size() * (sizeof(PromptMerge) / 4),
              words + items.size() * (sizeof(PromptItem) / 4));
  return TP_OK;
}

}  // namespace tp

using namespace tp;

extern "C" {

int tp_prompt_plan_make(const int64_t* q_lens, const int64_t* k_lens, int32_t n_seqs, int32_t num_q_heads,
                        int32_t num_kv_heads, tp_prompt_plan* plan, int32_t* words, size_t n_words) {
  try {
    return make_plan(q_lens, k_lens, n_seqs, num_q_heads, num_kv_heads, plan, words, n_words);
  } catch (const std::exception&) {  // the lists of a batch that asks for more items than the host has memory for
    return fail(TP_ERR_CUDA, "tp_prompt_plan_make: out of host memory");
  }
}

int tp_prompt_attention(const tp_prompt_plan* plan, const int32_t* words, const tp_prompt_rows* rows, const void* q,
                        const void* k, const void* v, float scale, void* out, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (!plan || !rows) return fail(TP_ERR_INVALID, "tp_prompt_attention: NULL argument");
  if (rows->dtype != TP_F16 && rows->dtype != TP_BF16)
    return fail(TP_ERR_INVALID, "tp_prompt_attention: q, k and v must be float16 or bfloat16");
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(TP_ERR_INVALID, "attention scale must be positive");
  if (plan->q_tokens == 0) return TP_OK;
  if (!words || !q || !out) return fail(TP_ERR_INVALID, "tp_prompt_attention: NULL argument");
  if (uintptr_t(out) % 16) return fail(TP_ERR_INVALID, "tp_prompt_attention: out must be 16-byte aligned");
  if (!workspace || workspace_bytes < plan->workspace_bytes)
    return fail(TP_ERR_INVALID, "tp_prompt_attention: workspace too small (need " +
                                    std::to_string(plan->workspace_bytes) + " bytes)");
  const bool bf16 = rows->dtype == TP_BF16;
  PromptParams P;
  P.hq = plan->num_q_heads;
  P.hkv = plan->num_kv_heads;
  P.group = P.hq / P.hkv;
  P.tile_tokens = tile_tokens_of(P.group);
  int st = rows_map(&P.qmap, q, plan->q_tokens, P.hq, rows->q[0], rows->q[1], P.group, P.tile_tokens, bf16, "q");
  // Without keys nothing is loaded and the maps are not read.
  if (st == TP_OK && plan->k_tokens)
    st = rows_map(&P.kmap, k, plan->k_tokens, P.hkv, rows->k[0], rows->k[1], 1, kKeys, bf16, "k");
  if (st == TP_OK && plan->k_tokens)
    st = rows_map(&P.vmap, v, plan->k_tokens, P.hkv, rows->v[0], rows->v[1], 1, kKeys, bf16, "v");
  if (st != TP_OK) return st;
  P.items = reinterpret_cast<const PromptItem*>(words);
  P.merges = reinterpret_cast<const PromptMerge*>(P.items + plan->items);
  P.merged = plan->merges > 0;
  P.scale_log2 = scale * 1.4426950408889634f;
  P.q = static_cast<const uint16_t*>(q);
  P.k = static_cast<const uint16_t*>(k);
  P.v = static_cast<const uint16_t*>(v);
  P.q_t = rows->q[0], P.q_h = rows->q[1], P.k_t = rows->k[0], P.k_h = rows->k[1], P.v_t = rows->v[0], P.v_h = rows->v[1];
  P.out = static_cast<uint16_t*>(out);
  P.error = static_cast<int*>(workspace);
  P.rec_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256);
  const size_t slots_rows = (plan->workspace_bytes - 256) / (kD * sizeof(float) + sizeof(float2));
  P.rec_ml = reinterpret_cast<float2*>(P.rec_o + slots_rows * kD);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan->block_tokens > P.tile_tokens)
    return bf16 ? launch_prompt<true, true>(P, *plan, s) : launch_prompt<false, true>(P, *plan, s);
  return bf16 ? launch_prompt<true, false>(P, *plan, s) : launch_prompt<false, false>(P, *plan, s);
}

}  // extern "C"
