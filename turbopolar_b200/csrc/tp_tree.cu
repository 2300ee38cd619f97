// Attention of drafted tokens over the compressed cache, the dense tail and each other.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j)
// over every cached token (pages decoded to float16 keys and values as tp_decode_pages decodes
// them, then the tail) and the drafts d with mask[t][d].
//
// The T drafts times the G query heads of a KV head are the rows; up to 256 rows (two tiles of 128)
// share each decoded page, so a page is read and decoded once per KV head for T * G <= 256, where
// one single-token call per draft would stream it T times.  The steps of all (KV head, row group)
// segments -- pages, tail, tiles of 64 drafts -- form one flat list, cut into equal ranges, one per
// SM; rows of a segment that several CTAs worked on are merged by merge_pieces_kernel.
//
//   warps 0-3, 4-7   softmax, one row per thread (queries live in tensor memory as operand A)
//   warps 8-15       decode: 64 keys and values per step into a ring of 32 KB stages
//   warp 16          issues the products
//   warp 17          copies pages as they are stored into a ring of three (bulk copies)
//   warps 18, 19     complete the warpgroup (registers are moved per warpgroup)
//
// Time, 32 drafts x 4 heads over 32K tokens: 40.3 us, where the pages' bytes take 12.1.  No pipe is busy (issue slots
// 48%, shared memory 31%, special functions 26%, tensor 19%): a step is a chain of latencies of about 1,700 cycles
// (page wait, stage wait, loads, decode, proxy fence, arrival), which all eight decode warps go through for an eighth
// of the page each.  Sixteen warps on the same chain gained nothing; no other arrangement of eight was tried.
// 64 drafts over 128K: 186 us, of which the products take 84.
// Short contexts (100 tokens, 5 drafts: 10.2 us) are one CTA's chain of copy, decode, scores, weights and rows.
//
// With more than 128 rows the softmax warpgroups have a tile each; with fewer they take
// alternate steps of the one tile, each with its own running maximum, sum and accumulator, and
// merge at the segment's end.
//
// Float32 queries, tails and drafts (100 tokens, 5 drafts: 15.4 us; 32K x 32: 52.5 us, a page for one tile of rows instead
// of two) are split into two float16 parts (22 bits), so only the weights and the output are
// rounded to float16; rounded inputs had twice the error of a float32 computation on contexts of few tokens.
// The queries' second part takes the tensor memory of a second tile, a key's second part a row of its own.  A row of
// queries or keys is first brought into float16's range by a power of two of its own, taken out again of its scores
// (of a query row what lies under 2^-39 of its largest is lost); scores of keys beyond 2^16 are made in float32.
// Values keep their size (under 1/4 their two parts are exact to 2^-25, as fine as the output's own last bit); rows with
// values beyond float16 stay out of the product and are added in float32 at the end, as rows of infinities are.
#include <algorithm>
#include <cmath>
#include <string>

#include "tp_codec.cuh"
#include "tp_umma.cuh"

namespace tp {

constexpr int kTreeKeys = 64;                         // keys per step: one page
constexpr int kKvHalf = kTreeKeys * 128;              // 64 keys x 64 channels
constexpr int kTreeStage = 4 * kKvHalf;               // K then V
constexpr int kTreeStages = 4;
constexpr int kPageRing = 3, kPageSlot = 2 * kMaxUnitBytes;  // stored pages on their way
constexpr int kPageCopiers = 4;
constexpr int kMaxDrafts = 256;
// Up to so many steps a CTA takes a whole segment: a second kernel costs about what four steps do.
constexpr int kWholeSteps = 4;
constexpr int kGroupRows = 2 * kTile;                 // rows that share a decoded page, at most
constexpr int kLateRing = 16;                         // segments whose lists may be alive
constexpr int kLateWords = 10;                        // a bit per draft, then per row of the tail
constexpr int kTreeThreads = 640;
// Five warpgroups at 96 registers: 480, of which the softmax threads take 128, decode 88, issue 48.
constexpr int kTreeSoftmaxRegs = 128, kTreeDecodeRegs = 88, kTreeIssueRegs = 48;
constexpr int kOffPages = kTreeStages * kTreeStage;
constexpr int kOffBits = kOffPages + kPageRing * kPageSlot;  // [2][128][4] uint64: drafts that a row sees
constexpr int kOffTab = kOffBits + 2 * 128 * 4 * 8;   // float2[512]
constexpr int kOffMl = kOffTab + 512 * 8;             // [2 pieces][2 warpgroups][128] float2
constexpr int kOffBuf = kOffMl + 2 * 2 * 128 * 8;     // 2 KB per softmax warp: rows on their way in and out
constexpr int kOffLate = kOffBuf + 8 * kStageRows;    // [kLateRing][kLateWords]
constexpr int kOffFactors = kOffLate + kLateRing * kLateWords * 4;  // [kTreeStages][32] float: of float32 keys
constexpr int kOffTreeBars = kOffFactors + kTreeStages * 32 * 4;
constexpr int kTreeSmem = kOffTreeBars + 256;

// Tensor memory (a CTA holds all of it): queries of tile t at 64 t, accumulator and scores t at
constexpr uint32_t kTreeOutCol = 128, kTreeScoreCol = 384;  // + 128 t and + 64 t

enum { kTreeDefault = 0, kTreeAdapter = 1, kTreeGeneral = 2 };

struct TreeParams {
  PoolArgs pool;
  const void *tail_k, *tail_v;
  int tail_f32, q_f32, kv_f32;
  int heads, hkv, hq, group, drafts, rows;  // heads: batch * hkv; rows: drafts * group
  int group_rows;                           // kGroupRows, or one tile
  int row_groups, n_page_steps, tail_len, n_tail_steps, n_steps, visible;
  int total, grid;                          // segments * n_steps; CTAs
  int merged;                               // merge_pieces_kernel follows
  float scale_log2;
  const void *q, *k, *v;
  int64_t q_b, q_h, q_t, k_b, k_h, k_t, v_b, v_h, v_t;
  const uint8_t* mask;
  int64_t mask_b, mask_t;
  __half* out;                              // [batch][drafts][hq][128]
  float* rec_o;                             // [piece][32][record rows][4]: channel / 4, row
  float2* rec_ml;
  int rec_rows;
  int* error;
  int32_t* d_state;                         // the cache's state words, or NULL
  int n_pages, state_tail, seq_len;         // what its first three are while this call's sizes hold
};
// (cos, sin) of the level-1 codes, then of the deep codes; of the 16 codes of both for the default format.
template <int kMode>
struct TreeAngles {
  float2 cs[kMode == kTreeDefault ? 16 : 512];
};

// False once the cache has changed since the call was made (a graph replayed after an append or a reset): its sizes
// and buffers are then another's, and nothing of it may be read.
__device__ __forceinline__ bool cache_as_called(const TreeParams& P) {
  if (!P.d_state) return true;
  const int pages = P.d_state[0], tail = P.d_state[1], tokens = P.d_state[2];  // three loads in flight
  return ((pages ^ P.n_pages) | (tail ^ P.state_tail) | (tokens ^ P.seq_len)) == 0;
}
// NaN rows instead of outputs.
__device__ __forceinline__ void refuse_rows(const TreeParams& P) {
  const uint32_t nan2 = 0x7fff7fffu;
  const int64_t chunks = int64_t(P.heads / P.hkv) * P.drafts * P.hq * (kD / 8);
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < chunks; i += int64_t(gridDim.x) * blockDim.x)
    reinterpret_cast<uint4*>(P.out)[i] = make_uint4(nan2, nan2, nan2, nan2);
  if (blockIdx.x == 0 && threadIdx.x == 0) P.d_state[4] = 4;
}

__device__ __forceinline__ int range_begin(const TreeParams& P, int cta) {
  return int(uint64_t(uint32_t(P.total)) * uint32_t(cta) / uint32_t(P.grid));
}
// The CTA whose range holds step f of the flat list.
__device__ __forceinline__ int range_of(const TreeParams& P, int f) {
  int cta = int(uint64_t(uint32_t(f)) * uint32_t(P.grid) / uint32_t(P.total));
  while (range_begin(P, cta + 1) <= f) ++cta;
  return cta;
}

// Unit layout of the two specialised formats: offsets known to the compiler become part of the load
// instructions.
template <int kMode>
struct UnitOf {
  static constexpr int vcodes = kMode == kTreeDefault ? 4096 : 2048, codes = vcodes + 4096,
                       vscales = codes + (kMode == kTreeDefault ? 1024 : 2048), bytes = vscales + 256;
};

// Decode thread tid takes pairs [8c, 8c + 8) of row l of both units; its warp, steps kk = 0, 1 (16 tokens)
// x 32 channels of group G of unit vu.  Eight neighbouring lanes hold four c of two rows: their chunks of
// a K tile lie in different banks.
struct DecodeShare {
  int c, l, G, vu, lane;
  __device__ __forceinline__ explicit DecodeShare(int tid)
      : c((tid & 3) | (tid >> 3 & 1) << 2), l((tid >> 2 & 1) | (tid >> 4) << 1), G(tid >> 5 & 3), vu(tid >> 7),
        lane(tid & 31) {}
};

__device__ __forceinline__ void st16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}

// The 16 channels of 8 decoded pairs of row `row`: two 16-byte chunks.
__device__ __forceinline__ void store_pairs(uint32_t k_tile, int row, int c, const uint32_t (&w)[8]) {
  const uint32_t base = k_tile + (c >> 2) * kKvHalf + row * 128;
  const int c0 = (2 * c) & 7;
  st16(base + ((c0 ^ (row & 7)) << 4), w[0], w[1], w[2], w[3]);
  st16(base + (((c0 + 1) ^ (row & 7)) << 4), w[4], w[5], w[6], w[7]);
}

// Decode the stored page at `pg` (shared memory) into the stage (K tile, V tile).  `limit`: tokens of
// the page that are seen; values of the others are cleared (their weights are 0, and 0 times a
// non-finite value is NaN).  `rscale`: the page's radius scale (int8 radii).
template <int kMode>
__device__ __forceinline__ void decode_step(const uint8_t* pg, const PoolArgs& L, const float2* tab, float rscale,
                                            uint32_t stage, int limit, int tid) {
  const DecodeShare D(tid);
  const int c = D.c, l = D.l;
  const int ub = kMode == kTreeGeneral ? L.unit_bytes : UnitOf<kMode>::bytes;
  const int vc = kMode == kTreeGeneral ? L.u_vcodes : UnitOf<kMode>::vcodes;
  const int vs = kMode == kTreeGeneral ? L.u_vscales : UnitOf<kMode>::vscales;
  uint32_t w[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const uint8_t* un = pg + u * ub;
    if (kMode == kTreeDefault) {
      // r (cos, sin) in float16 pairs with the cosine and sine as sums of two float16 numbers (an error
      // of 2^-22): r lo, then r hi + that, is the float32 product rounded once but for rare ties.  Half the
      // instructions of the float32 form; the decode warps' instructions bound this kernel.
      const uint4 rad = *reinterpret_cast<const uint4*>(un + radii_f16_offset(l, 8 * c));
      const uint32_t code = *reinterpret_cast<const uint32_t*>(un + UnitOf<kMode>::codes + l * 32 + 4 * c);
      const uint32_t rr[4] = {rad.x, rad.y, rad.z, rad.w};
      const uint32_t even = code << 3 & 0x78787878u, odd = code >> 1 & 0x78787878u;  // bytes: 8 * code
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t at = prmt(i & 1 ? odd : even, 0, 0x4440 + (i >> 1));
        const uint2 cs = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(tab) + at);
        const __half2 r2 = u32_as_h2(rr[i >> 1]), r = i & 1 ? __high2half2(r2) : __low2half2(r2);
        w[u][i] = h2_as_u32(__hfma2(r, u32_as_h2(cs.x), __hmul2(r, u32_as_h2(cs.y))));
      }
    } else if (kMode == kTreeAdapter) {
      const uint2 rad = *reinterpret_cast<const uint2*>(un + l * 64 + 8 * c);
      const uint2 code = *reinterpret_cast<const uint2*>(un + UnitOf<kMode>::codes + l * 64 + 8 * c);
      const float s = rscale * 1.4426950408889634f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t rw = i < 4 ? rad.x : rad.y, cw = i < 4 ? code.x : code.y;
        const float2 cs = tab[256 + ((cw >> (8 * (i & 3))) & 255)];
        const float r = exp2_approx(float(int8_t(rw >> (8 * (i & 3)))) * s);
        w[u][i] = pack_h2(r * cs.x, r * cs.y);
      }
    } else {
      const uint8_t* row = un + L.u_codes + l * L.code_row;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = 8 * c + i;
        const bool l1 = j < L.l1_pairs;
        const int rel = l1 ? j : j - L.l1_pairs, bits = l1 ? L.l1_bits : L.deep_bits;
        const int at = rel * bits;
        const uint32_t code = (row[(l1 ? 0 : L.l1_row) + (at >> 3)] >> (at & 7)) & ((1u << bits) - 1);
        const float r = L.int8_radii
                            ? exp2_approx(float(reinterpret_cast<const int8_t*>(un)[l * 64 + j]) * rscale * 1.4426950408889634f)
                            : __half2float(*reinterpret_cast<const __half*>(un + radii_f16_offset(l, j)));
        const float2 cs = tab[(l1 ? 0 : 256) + code];
        w[u][i] = pack_h2(r * cs.x, r * cs.y);
      }
    }
  }
  // Values: byte x of a word is code + 128; 0x6400 | x is the float16 number 1024 + x.
  const uint32_t v_tile = stage + 2 * kKvHalf;
  const int G = D.G, g = D.lane >> 2, t = D.lane & 3, chunk = (G & 1) * 4 + (g >> 1);
  const __half2 bias = __float2half2_rn(1152.0f);
  uint32_t o[2][4][2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    const uint4 v = *reinterpret_cast<const uint4*>(pg + D.vu * ub + vc + G * 512 + D.lane * 16 + kk * 2048);
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const __half2 sc = *reinterpret_cast<const __half2*>(pg + D.vu * ub + vs + (t * 16 + G * 2) * 2 + kk * 128 + a * 16);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const __half2 s2 = b ? __high2half2(sc) : __low2half2(sc);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          o[kk][2 * a + b][e] =
              h2_as_u32(__hmul2(__hsub2(u32_as_h2(prmt(words[2 * a + e], 0x64646464u, b ? 0x4341u : 0x4240u)), bias), s2));
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) store_pairs(stage, u * 32 + l, c, w[u]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int in_page = D.vu * 32 + (i >> 2) * 16 + (i >> 1 & 1) * 8 + 2 * t + (i & 1);
    st8(v_tile + (G >> 1) * kKvHalf + in_page * 128 + ((chunk ^ (in_page & 7)) << 4) + (g & 1) * 8, o[i >> 2][i & 3][0],
        o[i >> 2][i & 3][1]);
  }
  if (limit < kTreeKeys) {  // this thread's values again, where they are not seen
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int in_page = D.vu * 32 + (i >> 2) * 16 + (i >> 1 & 1) * 8 + 2 * t + (i & 1);
      if (in_page >= limit)
        st8(v_tile + (G >> 1) * kKvHalf + in_page * 128 + ((chunk ^ (in_page & 7)) << 4) + (g & 1) * 8, 0, 0);
    }
  }
}

__device__ __forceinline__ bool chunk_not_finite(uint4 x) {  // an exponent of all ones: one more carries over
  auto carry = [](uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; };
  return (carry(x.x) | carry(x.y) | carry(x.z) | carry(x.w)) & 0x80008000u;
}

// Eight float32 channels of a row.
struct Chunk32 {
  float4 a, b;
  __device__ __forceinline__ Chunk32() : a(make_float4(0.f, 0.f, 0.f, 0.f)), b(a) {}
  __device__ __forceinline__ Chunk32(const void* p, int64_t at)
      : a(*reinterpret_cast<const float4*>(static_cast<const float*>(p) + at)),
        b(*reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4)) {}
  __device__ __forceinline__ void scale(float f) {
    a.x *= f, a.y *= f, a.z *= f, a.w *= f, b.x *= f, b.y *= f, b.z *= f, b.w *= f;
  }
  __device__ __forceinline__ uint32_t top() const {  // bits of the largest finite magnitude, which order as numbers do
    auto finite = [](float x) {
      const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
      return u < 0x7f800000u ? u : 0u;
    };
    return max(max(max(finite(a.x), finite(a.y)), max(finite(a.z), finite(a.w))),
               max(max(finite(b.x), finite(b.y)), max(finite(b.z), finite(b.w))));
  }
};
// The power of two that brings a row whose largest magnitude has the bits `top` to [2^14, 2^15), at most 2^24: a row
// of at least 2^-27 keeps 22 bits, a smaller one 2^-49.  And its inverse.
__device__ __forceinline__ float row_factor(uint32_t top) {
  return top ? __uint_as_float(uint32_t(127 + min(24, 14 + 127 - int(top >> 23))) << 23) : 1.0f;
}
constexpr uint32_t kBeyondHalf = 0x47800000u;  // 2^16
__device__ __forceinline__ float inverse_factor(float f) { return __uint_as_float((254u << 23) - __float_as_uint(f)); }

// Two float16 parts: what the first rounds away is the second (nothing where the first is not finite).
__device__ __forceinline__ void split_chunk(const Chunk32& x, uint4& hi, uint4& lo) {
  const float4 &a = x.a, &b = x.b;
  auto rest = [](uint32_t h, float x, float y) {
    const float2 f = __half22float2(u32_as_h2(h));
    return pack_h2(isfinite(f.x) ? x - f.x : 0.0f, isfinite(f.y) ? y - f.y : 0.0f);
  };
  hi = make_uint4(pack_h2(a.x, a.y), pack_h2(a.z, a.w), pack_h2(b.x, b.y), pack_h2(b.z, b.w));
  lo = make_uint4(rest(hi.x, a.x, a.y), rest(hi.y, a.z, a.w), rest(hi.z, b.x, b.y), rest(hi.w, b.z, b.w));
}

// Float32 keys and values take two rows of the stage each, r and r + 32 (see split_chunk), so a step holds 32:
// scores of both rows are added, and the weight is written for both.
__host__ __device__ __forceinline__ int dense_keys(int f32) { return f32 ? kTreeKeys / 2 : kTreeKeys; }

// Rows [0, valid) of dense keys and values (row strides kt, vt) into the stage, the rest cleared.
// With `late`, a row with a value that is not finite as float16 sets its bit there; of float32 it is cleared, too.
// `factors`: where the scores' factors of float32 keys go, 0 for a key beyond float16.  All 256 decode threads.
__device__ __forceinline__ void dense_step(uint32_t stage, const void* k, const void* v, int64_t kt, int64_t vt, int f32,
                                           int valid, uint32_t* late, float* factors, int tid) {
  const int c = tid & 15;
  uint4 x[4], y[4];  // all loads in flight before the first is looked at
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = y[i] = make_uint4(0, 0, 0, 0);
  if (f32) {
    Chunk32 key[2], value[2];
    uint32_t top[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = i * 16 + (tid >> 4);
      if (row < valid) key[i] = Chunk32(k, row * kt + 8 * c), value[i] = Chunk32(v, row * vt + 8 * c);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) top[i] = key[i].top();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {  // 16 lanes to a row
#pragma unroll
      for (int i = 0; i < 2; ++i) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = i * 16 + (tid >> 4);
      const bool beyond = top[i] >= kBeyondHalf;
      if (beyond) key[i] = Chunk32();
      const float f = row_factor(top[i]);
      key[i].scale(f);
      split_chunk(key[i], x[i], x[i + 2]);
      split_chunk(value[i], y[i], y[i + 2]);
      const uint32_t listed = __ballot_sync(0xffffffffu, chunk_not_finite(y[i])) >> (tid & 16) & 0xffffu;
      if (listed) y[i] = y[i + 2] = make_uint4(0, 0, 0, 0);
      if (c == 0) {
        factors[row] = beyond ? 0.0f : inverse_factor(f);
        if (listed) atomicOr(late, 1u << row);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 16 + (tid >> 4);
      if (row < valid) {
        x[i] = *reinterpret_cast<const uint4*>(static_cast<const __half*>(k) + row * kt + 8 * c);
        y[i] = *reinterpret_cast<const uint4*>(static_cast<const __half*>(v) + row * vt + 8 * c);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 16 + (tid >> 4);
    const uint32_t at = stage + tile_chunk(row, c, kTreeKeys);
    st16(at, x[i].x, x[i].y, x[i].z, x[i].w);
    st16(at + 2 * kKvHalf, y[i].x, y[i].y, y[i].z, y[i].w);
    if (!f32 && late && chunk_not_finite(y[i])) atomicOr(late + (row >> 5), 1u << (row & 31));
  }
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int f32) {
  return f32 ? static_cast<const float*>(p)[i] : __half2float(static_cast<const __half*>(p)[i]);
}

// kPair: a tile per softmax warpgroup (more than 128 rows).
// kF32: the query, the tail or the drafts are float32 (an instance of its own: float16 calls were 4% slower in one).
template <int kMode, bool kPair, bool kF32>
__global__ void __launch_bounds__(kTreeThreads, 1) tree_attention_kernel(const __grid_constant__ TreeParams P,
                                                                          const __grid_constant__ TreeAngles<kMode> A) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int q_f32 = kF32 ? P.q_f32 : 0, kv_f32 = kF32 ? P.kv_f32 : 0, tail_f32 = kF32 ? P.tail_f32 : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2* tab = reinterpret_cast<float2*>(smem + kOffTab);
  uint32_t* late_ring = reinterpret_cast<uint32_t*>(smem + kOffLate);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + kOffTreeBars);
  uint64_t *kv_empty = kv_full + kTreeStages, *s_full = kv_empty + kTreeStages, *p_full = s_full + 2,
           *o_done = p_full + 2, *page_full = o_done + 2, *page_empty = page_full + kPageRing,
           *q_full = page_empty + kPageRing, *met = q_full + 1, *scanned = met + 1, *drained = scanned + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* stop = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* current = stop + 1;
  // One thread of a warp that sets up nothing else: 0.2 us, by all threads 0.5 us.
  if (threadIdx.x == 18 * 32) *current = cache_as_called(P);

  // (cos, sin) of every code; for the default format's 16 codes as float16 pairs, rounded and remainder.
  for (int i = threadIdx.x; i < int(sizeof(A.cs) / sizeof(float2)); i += kTreeThreads) {
    const float2 cs = A.cs[i];
    if (kMode == kTreeDefault) {
      const __half2 hi = __floats2half2_rn(cs.x, cs.y);
      const __half2 lo = __floats2half2_rn(cs.x - __low2float(hi), cs.y - __high2float(hi));
      reinterpret_cast<uint2*>(tab)[i] = make_uint2(h2_as_u32(hi), h2_as_u32(lo));
    } else {
      tab[i] = cs;
    }
  }
  for (int i = threadIdx.x; i < kLateRing * kLateWords; i += kTreeThreads) late_ring[i] = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kTreeStages; ++i) {
      mbar_init(kv_full + i, 8);
      mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 2);
      mbar_init(p_full + i, 4);
      mbar_init(o_done + i, 1);
    }
    for (int i = 0; i < kPageRing; ++i) {
      mbar_init(page_full + i, kPageCopiers);
      mbar_init(page_empty + i, 8);
    }
    mbar_init(q_full, 8);
    mbar_init(met, 8);
    mbar_init(scanned, 8);
    mbar_init(drained, 1);
    *stop = 0;
    fence_mbar_init();
  }
  if (warp == 16) tmem_alloc(tmem_slot, 512);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  // merge_pieces_kernel waits for this grid itself; nothing else may start before it has completed.
  if (P.merged) asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t tmem = *tmem_slot;
  if (tmem != 0 && threadIdx.x == 0) *stop = 1;  // all 512 columns: always at 0
  const int f0 = range_begin(P, blockIdx.x), count = *current ? range_begin(P, blockIdx.x + 1) - f0 : 0;
  const int seg0 = f0 / P.n_steps, step0 = f0 - seg0 * P.n_steps;
  const int draft0 = P.n_page_steps + P.n_tail_steps;  // first step of draft tiles

  if (warp < 8) {
    more_registers<kTreeSoftmaxRegs>();
    const int w = warp >> 2;
    const int r0 = (warp & 3) * 32 + lane;          // row in the tile
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_addr = kTreeScoreCol + 64 * w + lanes;
    uint64_t* bits = reinterpret_cast<uint64_t*>(smem + kOffBits) + (w * 128 + r0) * 4;
    float2* ml = reinterpret_cast<float2*>(smem + kOffMl);
    uint8_t* buf = smem + kOffBuf + warp * kStageRows;
    int units = 0, piece = 0, draft_pieces = 0;
    bool ok = true;
    for (int done = 0, seg = seg0, a = step0; done < count && ok; ++piece, ++seg, a = 0) {
      const int b = min(P.n_steps, a + count - done);
      const int head = seg / P.row_groups, rg = seg - head * P.row_groups;
      const int batch = head / P.hkv, kvh = head - batch * P.hkv;
      const int r = rg * P.group_rows + (kPair ? w * kTile : 0) + r0;
      const bool valid = r < P.rows;
      const int g = valid ? r / P.drafts : 0, t = valid ? r - g * P.drafts : 0;
      const int64_t q_at = batch * P.q_b + (int64_t(kvh) * P.group + g) * P.q_h + t * P.q_t;
      float q_factor = 1.0f, row_scale = P.scale_log2;
      if (!kPair && q_f32) {
        // Four lanes to a row here too.  Both warpgroups need the rows' factors, the first writes the queries: its
        // second parts to the columns of the second tile's.
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = 8 * i + (lane >> 2);
          const int64_t at = __shfl_sync(0xffffffffu, q_at, from);
          const bool there = __shfl_sync(0xffffffffu, int(valid), from);
          uint32_t top = 0;
#pragma unroll
          for (int p = 0; p < 4; ++p)
            if (there) top = max(top, Chunk32(P.q, at + 32 * p + 8 * (lane & 3)).top());
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          f[i] = row_factor(max(top, __shfl_xor_sync(0xffffffffu, top, 2)));
          const float own = __shfl_sync(0xffffffffu, f[i], 4 * (lane & 7));
          if (lane >> 3 == i) q_factor = own;
        }
        row_scale *= inverse_factor(q_factor);
#pragma unroll 1
        for (int p = 0; w == 0 && p < 4; ++p) {
          uint4 parts[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int from = 8 * i + (lane >> 2);
            const int64_t at = __shfl_sync(0xffffffffu, q_at, from);
            Chunk32 x;
            if (__shfl_sync(0xffffffffu, int(valid), from)) x = Chunk32(P.q, at + 32 * p + 8 * (lane & 3));
            x.scale(f[i]);
            split_chunk(x, parts[0][i], parts[1][i]);
          }
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *staged(buf, 8 * i + (lane >> 2), lane & 3) = parts[part][i];
            __syncwarp();
            uint32_t y[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 v = *staged(buf, lane, i);
              y[4 * i] = v.x, y[4 * i + 1] = v.y, y[4 * i + 2] = v.z, y[4 * i + 3] = v.w;
            }
            __syncwarp();
            tmem_st16(64 * part + lanes + 16 * p, y);
          }
        }
        tmem_wait_st();
      } else if (kPair || w == 0) {
        // Four lanes to a row, all loads in flight, then 64 bytes of every row at a time through `buf`.
        uint4 x[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = 8 * i + (lane >> 2);
          const int64_t at = __shfl_sync(0xffffffffu, q_at, from);
          const bool there = __shfl_sync(0xffffffffu, int(valid), from);
#pragma unroll
          for (int p = 0; p < 4; ++p)
            x[i][p] = there ? *reinterpret_cast<const uint4*>(static_cast<const __half*>(P.q) + at + 32 * p + 8 * (lane & 3))
                            : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *staged(buf, 8 * i + (lane >> 2), lane & 3) = x[i][p];
          __syncwarp();
          uint32_t y[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = *staged(buf, lane, i);
            y[4 * i] = v.x, y[4 * i + 1] = v.y, y[4 * i + 2] = v.z, y[4 * i + 3] = v.w;
          }
          __syncwarp();
          tmem_st16(64 * w + lanes + 16 * p, y);
        }
        tmem_wait_st();
      }
      if (b > draft0) {  // which drafts this row sees
        const uint8_t* m = P.mask + batch * P.mask_b + t * P.mask_t;
        for (int d0 = 0; d0 < P.drafts; d0 += 64) {
          uint64_t x = 0;
          const int n = min(64, P.drafts - d0);
          if ((uintptr_t(m) & 3) == 0) {
            // Four bytes at a time: bit 0 of a byte says whether it is not 0, and the product moves byte i to bit 28 + i.
            uint32_t word[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              word[i] = 4 * i + 3 < n ? *reinterpret_cast<const uint32_t*>(m + d0 + 4 * i) : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t set = (((word[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | word[i]) >> 7 & 0x01010101u;
              x |= uint64_t(set * 0x10204080u >> 28) << (4 * i);
            }
            for (int d = n & ~3; d < n; ++d) x |= uint64_t(m[d0 + d] != 0) << d;
          } else {
#pragma unroll 16
            for (int d = 0; d < n; ++d) x |= uint64_t(m[d0 + d] != 0) << d;
          }
          bits[d0 >> 6] = x;
        }
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      const bool live = __any_sync(0xffffffffu, valid);
      SoftmaxRow row;
      bool any = false;
      for (int s = a; s < b && ok; ++s) {
        if (!kPair && ((done + s - a) & 1) != w) continue;
        ok = __all_sync(0xffffffffu, wait_bar(s_full + w, units & 1, stop));
        if (ok && live) {
          tmem_fence_after();
          uint64_t sees = ~uint64_t(0);
          const bool twice = s >= draft0 ? kv_f32 : s >= P.n_page_steps && tail_f32;
          if (s >= draft0) {
            const int j = s - draft0;
            sees = twice ? bits[j >> 1] >> (32 * (j & 1)) | ~uint64_t(0) << 32 : bits[j];
          } else {
            const int n = s < P.n_page_steps ? P.visible - s * kTreeKeys
                                             : P.tail_len - (s - P.n_page_steps) * dense_keys(tail_f32);
            if (n < (twice ? 32 : kTreeKeys)) sees = ((uint64_t(1) << n) - 1) | (twice ? ~uint64_t(0) << 32 : 0);
          }
          const uint32_t o_addr = kTreeOutCol + 128 * w + lanes;
          auto before = [&] { return wait_bar(o_done + w, (units - 1) & 1, stop); };
          if (twice)
            ok = softmax_tile<kTreeKeys / 2, false, true>(
                row, s_addr, o_addr, Bits64{sees}, row_scale, !any, before,
                reinterpret_cast<const float*>(smem + kOffFactors) + 32 * ((done + s - a) & (kTreeStages - 1)), [&](int c) {
                  const bool draft = s >= draft0;
                  const float* k = draft ? static_cast<const float*>(P.k) + batch * P.k_b + kvh * P.k_h + (32 * (s - draft0) + c) * P.k_t
                                         : static_cast<const float*>(P.tail_k) + (int64_t(head) * kPage + 32 * (s - P.n_page_steps) + c) * kD;
                  float dot = 0.0f;
                  for (int i = 0; i < kD; ++i) dot = fmaf(load_any(P.q, q_at + i, q_f32), k[i], dot);
                  return dot * q_factor;
                });
          else
            ok = softmax_tile<kTreeKeys, false>(row, s_addr, o_addr, Bits64{sees}, row_scale, !any, before);
          tmem_fence_before();
        }
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(p_full + w);
        any = true;
        ++units;
      }
      if (ok && any) ok = __all_sync(0xffffffffu, wait_bar(o_done + w, (units - 1) & 1, stop));
      bool any0 = any, any1 = false;
      float2 other = make_float2(-INFINITY, 0.0f);
      if (!kPair && ok) {
        // Both warpgroups hold parts of the same rows: exchange maxima and sums, then each writes
        // half of the channels of both accumulators' weighted sum.
        float2* mine = ml + (piece & 1) * 256;
        mine[w * 128 + r0] = make_float2(row.ref, row.sum);
        __syncwarp();
        if (lane == 0) mbar_arrive(met);
        ok = __all_sync(0xffffffffu, wait_bar(met, piece & 1, stop));
        if (ok) other = mine[(w ^ 1) * 128 + r0];
        const int n = b - a, first = done & 1;  // warpgroup of the piece's first step
        any0 = n > 1 || first == 0;
        any1 = n > 1 || first == 1;
      }
      if (ok && live) {
        tmem_fence_after();
        const float ref0 = kPair || w == 0 ? row.ref : other.x, ref1 = kPair || w == 0 ? other.x : row.ref;
        const float top = fmaxf(row.ref, other.x);
        const float base = top == -INFINITY ? 0.0f : top;
        const float w0 = exp2_approx(ref0 - base), w1 = kPair ? 0.0f : exp2_approx(ref1 - base);
        const float sum = kPair ? row.sum
                                : w0 * (w == 0 ? row.sum : other.y) + w1 * (w == 0 ? other.y : row.sum);
        const bool whole = a == 0 && b == P.n_steps;
        const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t rec = int64_t(blockIdx.x) + seg;
        const int in_rec = r - rg * P.group_rows;
        const int64_t out_at = ((int64_t(batch) * P.drafts + t) * P.hq + int64_t(kvh) * P.group + g) * kD;
        uint8_t* dst = valid ? reinterpret_cast<uint8_t*>(P.out + out_at) : nullptr;
        const uint32_t* late = late_ring + (draft_pieces & (kLateRing - 1)) * kLateWords;
        bool listed = false;
        if (b > draft0)
          for (int i = 0; i < (P.drafts + 31) >> 5; ++i) listed |= late[i] != 0;
        const bool tail_listed = tail_f32 && b > P.n_page_steps && (late[8] | late[9]);
        const int c_begin = kPair ? 0 : 64 * w, c_end = kPair ? kD : 64 * w + 64;
        const uint32_t o0 = kTreeOutCol + (kPair ? 128 * w : 0) + lanes, o1 = kTreeOutCol + 128 + lanes;
#pragma unroll 1
        for (int c = c_begin; c < c_end; c += 32) {
          float o[32], x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.0f;
          if (any0) {
            tmem_ld32(o0 + c, o);
            tmem_wait_ld<32>(o);
            if (!kPair) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= w0;
            }
          }
          if (!kPair && any1) {
            tmem_ld32(o1 + c, x);
            tmem_wait_ld<32>(x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = fmaf(w1, x[i], o[i]);
          }
          if (valid) {
            if (listed) {  // drafts with non-finite values that this row sees
              for (int d = 0; d < P.drafts; ++d) {
                if (!(late[d >> 5] >> (d & 31) & 1) || !(bits[d >> 6] >> (d & 63) & 1)) continue;
                const int64_t k_at = batch * P.k_b + kvh * P.k_h + d * P.k_t, v_at = batch * P.v_b + kvh * P.v_h + d * P.v_t;
                float dot = 0.0f;
                for (int i = 0; i < kD; ++i) dot = fmaf(load_any(P.q, q_at + i, q_f32), load_any(P.k, k_at + i, kv_f32), dot);
                const float p = exp2_approx(fmaf(dot, P.scale_log2, -base));
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = fmaf(p, load_any(P.v, v_at + c + i, kv_f32), o[i]);
              }
            }
            if (tail_listed) {  // and rows of the tail, which every row sees
              for (int d = 0; d < P.tail_len; ++d) {
                if (!(late[8 + (d >> 5)] >> (d & 31) & 1)) continue;
                const int64_t at = (int64_t(head) * kPage + d) * kD;
                const float *k = static_cast<const float*>(P.tail_k) + at, *v = static_cast<const float*>(P.tail_v) + at + c;
                float dot = 0.0f;
                for (int i = 0; i < kD; ++i) dot = fmaf(load_any(P.q, q_at + i, q_f32), k[i], dot);
                const float p = exp2_approx(fmaf(dot, P.scale_log2, -base));
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = fmaf(p, v[i], o[i]);
              }
            }
          }
          __syncwarp();
          if (whole) {
            uint32_t y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = pack_h2(o[2 * i] * inv, o[2 * i + 1] * inv);
            store_rows64(buf, y, dst ? dst + 2 * c : nullptr);
          } else {
            float4* to = reinterpret_cast<float4*>(P.rec_o) + (rec * 32 + c / 4) * P.rec_rows + in_rec;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (valid) to[i * P.rec_rows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          __syncwarp();
        }
        if (!whole && valid && (kPair || w == 0)) 
          P.rec_ml[rec * P.rec_rows + in_rec] = make_float2(kPair ? row.ref : top, sum);
      }
      tmem_fence_before();
      ++draft_pieces;
      done += b - a;
    }
  } else if (warp < 16) {
    fewer_registers<kTreeDecodeRegs>();
    const int tid = threadIdx.x - 256;
    const uint32_t stages = smem_u32(smem);
    int s = step0, seg = seg0, head = seg0 / P.row_groups;
    int st = 0, ph = 1, scans = 0, draft_pieces = 0;  // ph: parity of the stage's last release
    int slot = 0, slot_ph = 0;                        // page ring
    float rscale = 0.0f, rscale_next = 0.0f;
    auto radius_scale = [&](int h, int page) {
      return P.pool.int8_radii ? __half2float(P.pool.radii_scales[int64_t(h) * P.pool.page_capacity + page]) : 0.0f;
    };
    if (kMode != kTreeDefault && count && s < P.n_page_steps) rscale_next = radius_scale(head, s);
    bool ok = true;
    for (int i = 0; i < count && ok; ++i) {
      const int at = s, h = head;
      if (++s == P.n_steps) {
        s = 0;
        ++seg;
        head = seg / P.row_groups;
      }
      if (kMode != kTreeDefault) {
        rscale = rscale_next;
        if (i + 1 < count && s < P.n_page_steps) rscale_next = radius_scale(head, s);
      }
      const uint32_t stage = stages + st * kTreeStage;
      float* factors = reinterpret_cast<float*>(smem + kOffFactors) + 32 * st;
      ok = i < kTreeStages || warp_wait(kv_empty + st, ph, stop);
      if (!ok) break;
      if (at < P.n_page_steps) {
        ok = warp_wait(page_full + slot, slot_ph, stop);
        if (!ok) break;
        decode_step<kMode>(smem + kOffPages + slot * kPageSlot, P.pool, tab, rscale, stage, P.visible - at * kTreeKeys, tid);
        __syncwarp();
        if (lane == 0) mbar_arrive(page_empty + slot);
        if (++slot == kPageRing) slot = 0, slot_ph ^= 1;
      } else if (at < draft0) {
        const int t0 = (at - P.n_page_steps) * dense_keys(tail_f32);
        const int64_t row0 = (int64_t(h) * kPage + t0) * kD * (tail_f32 ? 4 : 2);
        dense_step(stage, static_cast<const uint8_t*>(P.tail_k) + row0, static_cast<const uint8_t*>(P.tail_v) + row0, kD, kD,
                   tail_f32, min(dense_keys(tail_f32), P.tail_len - t0),
                   tail_f32 ? late_ring + (draft_pieces & (kLateRing - 1)) * kLateWords + 8 + (t0 >> 5) : nullptr, factors, tid);
      } else {
        const int batch = h / P.hkv, kvh = h - batch * P.hkv, d0 = (at - draft0) * dense_keys(kv_f32);
        const int size = kv_f32 ? 4 : 2;
        uint32_t* late = late_ring + (draft_pieces & (kLateRing - 1)) * kLateWords;
        if (tid < kLateWords && (at == draft0 || i == 0))
          late_ring[((draft_pieces + kLateRing / 2) & (kLateRing - 1)) * kLateWords + tid] = 0;
        const int n = min(dense_keys(kv_f32), P.drafts - d0);
        dense_step(stage, static_cast<const uint8_t*>(P.k) + (batch * P.k_b + kvh * P.k_h + d0 * P.k_t) * size,
                   static_cast<const uint8_t*>(P.v) + (batch * P.v_b + kvh * P.v_h + d0 * P.v_t) * size, P.k_t, P.v_t,
                   kv_f32, n, late + (d0 >> 5), factors, tid);
        __syncwarp();
        if (lane == 0) mbar_arrive(scanned);
        ok = warp_wait(scanned, scans & 1, stop);
        if (!ok) break;
        ++scans;
        for (int q = 0; q < 4; ++q) {
          const int row = q * 16 + (tid >> 4), key = row & (dense_keys(kv_f32) - 1);
          if (late[(d0 >> 5) + (key >> 5)] >> (key & 31) & 1)
            st16(stage + 2 * kKvHalf + tile_chunk(row, tid & 15, kTreeKeys), 0, 0, 0, 0);
        }
        if (at == P.n_steps - 1) ++draft_pieces;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kv_full + st);
      if (++st == kTreeStages) st = 0, ph ^= 1;
    }
  } else if (fewer_registers<kTreeIssueRegs>(); warp == 16) {
    constexpr uint32_t kScores = mma_idesc(false, kTreeKeys, false), kOut = mma_idesc(false, kD, true);
    const uint32_t stages = smem_u32(smem);
    int n[2] = {0, 0};
    int st_s = 0, ph_s = 0, st_v = 0;  // ring: stage and phase of the next scores, stage of the next values
    bool ok = true;
    int a = step0;
    for (int done = 0, piece = 0; done < count && ok; ++piece, a = 0) {
      const int b = min(P.n_steps, a + count - done);
      const int n_units = (b - a) * (kPair ? 2 : 1);
      uint32_t acc[2] = {0, 0};
      ok = warp_wait(q_full, piece & 1, stop);
      // Unit u: (step, tile) pairs with two tiles, steps taking turns at the warpgroups with one.
      auto tile_of = [&](int u) { return kPair ? u & 1 : (done + u) & 1; };
      auto scores = [&](int u) {
        const int t = tile_of(u);
        if ((!kPair || t == 0) && !warp_wait(kv_full + st_s, ph_s, stop)) return false;
        tmem_fence_after();
        if (elect_one()) {
          const uint32_t k_lo = rows_lo(stages) + st_s * (kTreeStage >> 4);
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks)
            mma_ts(kTreeScoreCol + 64 * t, (kPair ? 64 * t : 0) + ks * 8, k_lo + (((ks >> 2) * kKvHalf + (ks & 3) * 32) >> 4),
                   kScores, ks > 0);
          if (!kPair && q_f32) {
#pragma unroll
            for (int ks = 0; ks < kD / 16; ++ks)
              mma_ts(kTreeScoreCol + 64 * t, 64 + ks * 8, k_lo + (((ks >> 2) * kKvHalf + (ks & 3) * 32) >> 4), kScores, true);
          }
          mbar_arrive(s_full + t);  // makes what this warp has acquired from the decode warps visible
          mma_commit(s_full + t);
        }
        __syncwarp();
        if (!kPair || t == 1) st_s = st_s + 1 == kTreeStages ? (ph_s ^= 1, 0) : st_s + 1;
        return true;
      };
      auto values = [&](int u) {
        const int t = tile_of(u);
        if (!warp_wait(p_full + t, (t ? n[1] : n[0]) & 1, stop)) return false;
        tmem_fence_after();
        if (elect_one()) {
          const uint32_t v_lo = cols_lo(stages + 2 * kKvHalf, kKvHalf) + st_v * (kTreeStage >> 4);
#pragma unroll
          for (int ks = 0; ks < kTreeKeys / 16; ++ks)
            mma_ts(kTreeOutCol + 128 * t, kTreeScoreCol + 64 * t + ks * 8, v_lo + ks * (2048 >> 4), kOut,
                   ks > 0 || (t ? acc[1] : acc[0]));
          mma_commit(o_done + t);
          if (!kPair || t == 1) mma_commit(kv_empty + st_v);
        }
        __syncwarp();
        if (t) acc[1] = 1, ++n[1];
        else acc[0] = 1, ++n[0];
        if (!kPair || t == 1) st_v = st_v + 1 == kTreeStages ? 0 : st_v + 1;
        return true;
      };
      if (ok) ok = scores(0) && (n_units < 2 || scores(1));
      for (int u = 0; u < n_units && ok; ++u) {
        ok = values(u);
        if (ok && u + 2 < n_units) ok = scores(u + 2);
      }
      done += b - a;
    }
    if (elect_one()) mma_commit(drained);
    __syncwarp();
    drain_bar(drained, 0);
    __syncwarp();
  } else if (warp == 17 && lane < kPageCopiers) {
    // Each of four lanes copies a quarter of every page (issuing a copy blocks a thread for some hundred
    // cycles; lanes dispatch in parallel).
    const uint32_t part = P.pool.page_bytes / kPageCopiers;
    const uint64_t policy = l2_evict_first_policy();
    int s = step0, seg = seg0, slot = 0, slot_ph = 1, issued = 0;
    for (int i = 0; i < count; ++i) {
      if (s < P.n_page_steps) {
        if (issued >= kPageRing && !wait_bar(page_empty + slot, slot_ph, stop)) break;
        const uint8_t* pg =
            P.pool.pages + (int64_t(seg / P.row_groups) * P.pool.page_capacity + s) * P.pool.page_bytes + lane * part;
        mbar_arrive_expect_tx(page_full + slot, part);
        bulk_g2s_hint(smem + kOffPages + slot * kPageSlot + lane * part, pg, part, page_full + slot, policy);
        ++issued;
        if (++slot == kPageRing) slot = 0, slot_ph ^= 1;
      }
      if (++s == P.n_steps) s = 0, ++seg;
    }
    // No copy may be in flight when the CTA ends.
    for (int i = max(0, issued - kPageRing); i < issued; ++i) drain_bar(page_full + i % kPageRing, (i / kPageRing) & 1);
  }
  __syncthreads();
  if (warp == 16) {
    tmem_fence_after();
    tmem_free(tmem, 512);
  }
  if (threadIdx.x == 0 && *stop) {
    *P.error = 1;
    if (P.d_state) P.d_state[4] = 3;
  }
  if (!*current) refuse_rows(P);
}

// Rows of segments that several CTAs worked on: 32 rows x 8 channels per block, or per warp where a
// segment has few records.
template <bool kFew>
__global__ void __launch_bounds__(kMergeThreads, kFew ? 2 : 4) merge_pieces_kernel(const __grid_constant__ TreeParams P) {
  const int seg = blockIdx.x, head = seg / P.row_groups, rg = seg - head * P.row_groups;
  const int i0 = blockIdx.y * 32, rows = min(32, min(P.group_rows, P.rows - rg * P.group_rows) - i0);
  const int part = kFew ? blockIdx.z * (kMergeThreads / 32) + (threadIdx.x >> 5) : blockIdx.z;  // channels 8 part ..
  const int lane = threadIdx.x & 31;
  // CTAs whose ranges meet the segment's steps.
  const int first = range_of(P, seg * P.n_steps), last = range_of(P, (seg + 1) * P.n_steps - 1);
  const bool as_called = cache_as_called(P);  // nothing changes it before this call has ended
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (rows <= 0 || first == last || !as_called) return;  // one CTA: it has written the rows
  const int64_t rec = int64_t(first) + seg;
  MergePart p;
  if (!merge_records<kFew>(p, P.rec_ml + rec * P.rec_rows + i0,
                           reinterpret_cast<const float4*>(P.rec_o) + (rec * 32 + 2 * part) * P.rec_rows + i0, P.rec_rows,
                           int64_t(32) * P.rec_rows, P.rec_rows, last - first + 1, rows) ||
      lane >= rows)
    return;
  const int r = rg * P.group_rows + i0 + lane;
  const int batch = head / P.hkv, kvh = head - batch * P.hkv, g = r / P.drafts, t = r - g * P.drafts;
  *reinterpret_cast<uint4*>(P.out + ((int64_t(batch) * P.drafts + t) * P.hq + int64_t(kvh) * P.group + g) * kD + 8 * part) =
      make_uint4(pack_h2(p.acc[0], p.acc[1]), pack_h2(p.acc[2], p.acc[3]), pack_h2(p.acc[4], p.acc[5]),
                 pack_h2(p.acc[6], p.acc[7]));
}

// ----------------------------------------------------------------------------- host
// (cos, sin) of every code of 2, 4 or 8 bits, the decoder's angle formula in float32 (rfsn_v11/quant/
// polar/decoder.py:36-56), cosine and sine rounded to float32; computed once.
static void copy_angles(float2* cs, int bits) {
  static float2 table[9][256];
  static std::once_flag once;
  std::call_once(once, [] {
    for (int b : {2, 4, 8}) {
      const int n = 1 << b;
      for (int code = 0; code < n; ++code) {
        const float norm = float(code) / float(n - 1);
        volatile float turned = norm * 6.28318530717958647692f;  // rounded before the subtraction
        const float angle = turned - 3.14159265358979323846f;
        table[b][code] = make_float2(float(std::cos(double(angle))), float(std::sin(double(angle))));
      }
    }
  });
  std::copy_n(table[bits], 1 << bits, cs);
}

template <int kMode, bool kPair, bool kF32>
static int launch_tree(const TreeParams& P, const tp_format& fmt, int segments, cudaStream_t s) {
  static bool allowed[64] = {};  // the attribute belongs to a device's copy of the kernel
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !allowed[dev])) {
    const int st = allow_kernel(reinterpret_cast<const void*>(tree_attention_kernel<kMode, kPair, kF32>), kTreeSmem, kTreeThreads,
                                2 * kTreeSoftmaxRegs + 2 * kTreeDecodeRegs + kTreeIssueRegs, "tp_tree_attention");
    if (st != TP_OK) return st;
    if (dev < 64) allowed[dev] = true;
  }
  if (e != cudaSuccess) return fail(TP_ERR_CUDA, std::string("tp_tree_attention: ") + cudaGetErrorString(e));
  TreeAngles<kMode> A;
  copy_angles(A.cs, fmt.l1_bits);
  if constexpr (kMode != kTreeDefault) copy_angles(A.cs + 256, fmt.deep_bits);
  tree_attention_kernel<kMode, kPair, kF32><<<P.grid, kTreeThreads, kTreeSmem, s>>>(P, A);
  if (P.merged) {
    const int blocks = (P.rec_rows + 31) / 32;
    const bool few = P.n_steps / (P.total / P.grid) + 2 <= kFewRecords;  // CTAs that can share a segment
    e = few ? launch_dependent(merge_pieces_kernel<true>, dim3(segments, blocks, kD / 8 / (kMergeThreads / 32)), kMergeThreads, s, P)
            : launch_dependent(merge_pieces_kernel<false>, dim3(segments, blocks, kD / 8), kMergeThreads, s, P);
    if (e != cudaSuccess) return fail(TP_ERR_CUDA, std::string("tp_tree_attention: ") + cudaGetErrorString(e));
  }
  return check_launch("tp_tree_attention");
}

template <int kMode>
static int launch_tree_rows(const TreeParams& P, const tp_format& fmt, int segments, cudaStream_t s) {
  const bool pair = P.rows > kTile && P.group_rows > kTile;
  if (P.q_f32 || P.kv_f32 || (P.tail_f32 && P.tail_len > 0))
    return pair ? launch_tree<kMode, true, true>(P, fmt, segments, s) : launch_tree<kMode, false, true>(P, fmt, segments, s);
  return pair ? launch_tree<kMode, true, false>(P, fmt, segments, s) : launch_tree<kMode, false, false>(P, fmt, segments, s);
}

static int row_groups_of(int64_t rows, int group_rows) { return int((rows + group_rows - 1) / group_rows); }

static size_t tree_workspace(int64_t heads, int64_t rows) {
  size_t need = 0;
  for (int group : {kTile, kGroupRows}) {  // by the queries' type
    const int64_t slots = heads * row_groups_of(rows, group) + device_sms();
    need = std::max(need, size_t(slots) * std::min<int64_t>(rows, group) * (kD * sizeof(float) + sizeof(float2)));
  }
  return 256 + need;
}

static bool rows_ok(const void* p, const int64_t* st, const int* n, int f32) {
  const int step = f32 ? 4 : 8;
  if (uintptr_t(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && st[i] % step) return false;
  return true;
}

}  // namespace tp

using namespace tp;

extern "C" {

size_t tp_tree_attention_workspace_size(int32_t num_kv_heads, int32_t num_q_heads, int32_t n_drafts) {
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || n_drafts < 1 || n_drafts > kMaxDrafts) return 0;
  return tree_workspace(num_kv_heads, int64_t(n_drafts) * (num_q_heads / num_kv_heads));
}

int tp_tree_attention(const tp_page_pool* pool, const tp_tail* tail, tp_state state, const tp_drafts* drafts,
                      const void* q, const void* k, const void* v, const void* mask, float scale, void* out,
                      void* workspace, size_t workspace_bytes, void* stream) {
  Layout L;
  int st = validate_pool(pool, &L);
  if (st != TP_OK) return st;
  if (!drafts || !q || !k || !v || !mask || !out) return fail(TP_ERR_INVALID, "tp_tree_attention: NULL argument");
  const tp_drafts& D = *drafts;
  const int heads = pool->num_kv_heads;
  if (D.batch < 1 || heads % D.batch) return fail(TP_ERR_INVALID, "tp_tree_attention: batch does not divide the pool's heads");
  const int hkv = heads / D.batch;
  if (D.num_q_heads < 1 || D.num_q_heads % hkv)
    return fail(TP_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads for GQA");
  if (D.n_drafts < 1 || D.n_drafts > kMaxDrafts)
    return fail(TP_ERR_INVALID, "tp_tree_attention: n_drafts must be in [1, 256]");
  if ((D.q_dtype != TP_F16 && D.q_dtype != TP_F32) || (D.kv_dtype != TP_F16 && D.kv_dtype != TP_F32))
    return fail(TP_ERR_INVALID, "tp_tree_attention: q, k and v must be float16 or float32");
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(TP_ERR_INVALID, "attention scale must be positive");
  if (state.n_pages < 0 || state.n_pages > pool->page_capacity || state.tail_len < 0 || state.tail_len >= kPage ||
      state.first_page != 0)
    return fail(TP_ERR_INVALID, "tp_tree_attention: cache state outside the pool, or a sequence shard");
  const int64_t cached = int64_t(state.n_pages) * kPage + state.tail_len;
  if (state.seq_len < 0 || state.seq_len > cached)
    return fail(TP_ERR_INVALID, "tp_tree_attention: seq_len outside the cached tokens");
  if (state.tail_len > 0 && (!tail || !tail->k || !tail->v || (uintptr_t(tail->k) | uintptr_t(tail->v)) % 16))
    return fail(TP_ERR_INVALID, "tp_tree_attention: tail buffers missing");
  if (state.tail_len > 0 && tail->dtype != TP_F16 && tail->dtype != TP_F32)
    return fail(TP_ERR_INVALID, "tp_tree_attention: tail dtype must be float16 or float32");
  const int q_n[3] = {D.batch, D.num_q_heads, D.n_drafts}, kv_n[3] = {D.batch, hkv, D.n_drafts};
  if (!rows_ok(q, D.q, q_n, D.q_dtype == TP_F32) || !rows_ok(k, D.k, kv_n, D.kv_dtype == TP_F32) ||
      !rows_ok(v, D.v, kv_n, D.kv_dtype == TP_F32) || uintptr_t(out) % 16)
    return fail(TP_ERR_INVALID, "tp_tree_attention: rows must start on 16-byte boundaries");
  const int group = D.num_q_heads / hkv;
  const int64_t rows = int64_t(group) * D.n_drafts;
  const size_t need = tree_workspace(heads, rows);
  if (!workspace || workspace_bytes < need)
    return fail(TP_ERR_INVALID, "tp_tree_attention: workspace too small (need " + std::to_string(need) + " bytes)");

  TreeParams P;
  P.pool = pool_args(*pool, L);
  P.tail_k = tail ? tail->k : nullptr;
  P.tail_v = tail ? tail->v : nullptr;
  P.tail_f32 = tail && tail->dtype == TP_F32;
  P.q_f32 = D.q_dtype == TP_F32;
  P.kv_f32 = D.kv_dtype == TP_F32;
  P.heads = heads;
  P.hkv = hkv;
  P.hq = D.num_q_heads;
  P.group = group;
  P.drafts = D.n_drafts;
  P.rows = int(rows);
  // Float32 queries take two parts of tensor memory, so one tile of rows instead of two shares a page.
  P.group_rows = P.q_f32 ? kTile : kGroupRows;
  P.row_groups = row_groups_of(rows, P.group_rows);
  P.visible = int(std::min<int64_t>(state.seq_len, int64_t(state.n_pages) * kPage));
  P.n_page_steps = (P.visible + kPage - 1) / kPage;
  P.tail_len = int(std::max<int64_t>(0, state.seq_len - int64_t(state.n_pages) * kPage));
  auto steps_of = [](int keys, int f32) { return (keys + kTreeKeys / (f32 ? 2 : 1) - 1) / (kTreeKeys / (f32 ? 2 : 1)); };
  P.n_tail_steps = steps_of(P.tail_len, P.tail_f32);
  P.n_steps = P.n_page_steps + P.n_tail_steps + steps_of(D.n_drafts, P.kv_f32);
  const int64_t segments = int64_t(heads) * P.row_groups;
  const int64_t total = segments * P.n_steps;
  if (segments > (1 << 24) || total > (1 << 30))
    return fail(TP_ERR_UNSUPPORTED, "tp_tree_attention: too many heads, drafts or pages");
  // A CTA per segment where that is at most kWholeSteps steps: no second kernel.  Otherwise one CTA per SM.
  P.grid = int(P.n_steps <= kWholeSteps && segments <= device_sms() ? segments : std::min<int64_t>(device_sms(), total));
  P.total = int(total);
  P.merged = P.grid != segments;  // else each CTA has a segment to itself
  P.scale_log2 = scale * 1.4426950408889634f;
  P.q = q, P.k = k, P.v = v;
  P.q_b = D.q[0], P.q_h = D.q[1], P.q_t = D.q[2];
  P.k_b = D.k[0], P.k_h = D.k[1], P.k_t = D.k[2];
  P.v_b = D.v[0], P.v_h = D.v[1], P.v_t = D.v[2];
  P.mask = static_cast<const uint8_t*>(mask);
  P.mask_b = D.mask[0], P.mask_t = D.mask[1];
  P.out = static_cast<__half*>(out);
  P.error = static_cast<int*>(workspace);
  P.d_state = D.d_state;
  P.n_pages = state.n_pages, P.state_tail = state.tail_len, P.seq_len = state.seq_len;
  P.rec_rows = int(std::min<int64_t>(rows, P.group_rows));
  P.rec_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256);
  P.rec_ml = reinterpret_cast<float2*>(P.rec_o + (segments + device_sms()) * P.rec_rows * kD);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const tp_format& F = pool->fmt;
  if (F.l1_bits == 4 && F.deep_bits == 4 && F.split_dim == 64 && !F.int8_radii)
    return launch_tree_rows<kTreeDefault>(P, F, int(segments), s);
  if (F.int8_radii && F.split_dim == 0 && F.deep_bits == 8) return launch_tree_rows<kTreeAdapter>(P, F, int(segments), s);
  return launch_tree_rows<kTreeGeneral>(P, F, int(segments), s);
}

}  // extern "C"
