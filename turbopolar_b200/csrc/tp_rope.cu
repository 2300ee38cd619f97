// Norm of each query and key head and the position rotation, in one pass over the rows.
//
// For one row x of 128 channels (one token of one head) at angle rows c, s of its position:
//   y = x * rsqrt(mean(x^2) + eps) * w            (y = x without weights)
//   pairs (a, b) = (y[d], y[d + 64]), or (y[2d], y[2d + 1]) when interleaved, d = 0..63
//   out_a = a c[d] - b s[d],   out_b = b c[d] + a s[d]
// The row is read once, the sum of squares and the rotation are float32, and the result is rounded
// once to the output type.
//
// Bound: memory (read + write of q and k; 8,192 bfloat16 tokens of 32 + 8 heads move 172 MB).  A
// group of 16 lanes owns a row: lane i holds channels [4i, 4i+4) and [64+4i, 64+4i+4), so both
// pairings are inside one lane and only the sum of squares crosses lanes: for four rows at once in nine
// shuffles and one reciprocal root, where row by row takes sixteen and four.
//
// Measured, those 8,192 tokens: 29.7 us, 5.8 TB/s, where a copy of the size takes 26.6 us.  Issue slots are 60%
// used: a group's heads are all query or all key heads and sums and rotations are two float32 to an instruction,
// which took 36.6 us to that.  CTAs of 256 threads 31.2 us; bounds for ten or twelve CTAs per SM 31.5 and 40.6.
// Earlier and slower: groups of 8 lanes with 16-byte words (123 registers), two, five or eight heads per group.
// One token of 40 heads takes 1.9 us, 48 float32 tokens 2.5 us: launch latency.
#include <cuda_bf16.h>

#include "tp_umma.cuh"

namespace tp {

struct RopeSide {  // the query or the key heads
  const void* in;
  void* out;
  const void* weight;
  int64_t in_b, in_t, in_h, out_b, out_t, out_h;  // strides in elements
};

struct RopeParams {
  RopeSide q, k;
  const void *cos, *sin;
  const void* positions;
  int64_t table_stride, pos_b, pos_t;
  uint32_t n_units;     // batch * tokens * head groups
  uint32_t groups, q_groups;  // head groups of a token, and those of its query heads
  int batch, tokens, hq, hkv, table_rows, table_b_rows;
  int pos64, table_dtype, weight_dtype, interleaved;
  int table_words, weight_words;  // rows allow loads of four elements at a time
  float eps;
};

template <typename T> struct Pack4;  // four elements of a row, moved as one word
template <> struct Pack4<float> {
  float4 v;
  __device__ __forceinline__ void get(float* f) const { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
  __device__ __forceinline__ void set(const float* f) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Pack4<__half> {
  uint2 v;
  __device__ __forceinline__ void get(float* f) const {
    const float2 a = __half22float2(u32_as_h2(v.x)), b = __half22float2(u32_as_h2(v.y));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
  }
  __device__ __forceinline__ void set(const float* f) { v = make_uint2(pack_h2(f[0], f[1]), pack_h2(f[2], f[3])); }
};
template <> struct Pack4<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void get(float* f) const {
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
  __device__ __forceinline__ void set(const float* f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    v = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
};

// N (2 or 4) weights or angles from element i; `words`: N elements on their own boundary.
template <int N>
__device__ __forceinline__ void load_small(const void* p, int64_t i, int dtype, bool words, float* f) {
  if (dtype == TP_F32 && words) {
    const float* q = static_cast<const float*>(p) + i;
    if (N == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(q));
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
      const float2 v = __ldg(reinterpret_cast<const float2*>(q));
      f[0] = v.x, f[1] = v.y;
    }
    return;
  }
  if (words && N == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
    if (dtype == TP_F16) reinterpret_cast<const Pack4<__half>&>(v).get(f);
    else reinterpret_cast<const Pack4<__nv_bfloat16>&>(v).get(f);
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    f[j] = dtype == TP_F32   ? static_cast<const float*>(p)[i + j]
           : dtype == TP_F16 ? __half2float(static_cast<const __half*>(p)[i + j])
                             : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i + j]);
  }
}

// Many rows pass by once and are marked as the first to leave the L2 (8,192 tokens: 32.5 us without, 29.7 us
// with); the rows of a few tokens stay for whoever reads them next.
template <int kRows, typename T>
__device__ __forceinline__ auto load_row(const T* from) {
  const auto* p = &reinterpret_cast<const Pack4<T>*>(from)->v;
  return kRows > 1 ? __ldcs(p) : *p;
}
template <int kRows, typename T>
__device__ __forceinline__ void store_row(T* to, const Pack4<T>& x) {
  auto* p = &reinterpret_cast<Pack4<T>*>(to)->v;
  if (kRows > 1) __stcs(p, x.v);
  else *p = x.v;
}

__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {  // two float32 each
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// kRows query heads, or key heads, of one token per 16-lane group.
template <typename T, int kRows, bool kInterleaved>
__global__ void __launch_bounds__(128) norm_rope_kernel(const __grid_constant__ RopeParams P) {
  static_assert(kRows == 1 || kRows == 4, "the sums of squares are reduced for one row or four");
  const int lane = threadIdx.x & 15;
  const unsigned group_mask = 0xffffu << (threadIdx.x & 16);
  const uint32_t unit = blockIdx.x * (blockDim.x >> 4) + (threadIdx.x >> 4);
  if (unit >= P.n_units) return;
  const uint32_t row = unit / P.groups, hg = unit - row * P.groups;
  const bool is_q = hg < P.q_groups;
  const RopeSide& S = is_q ? P.q : P.k;
  const int h0 = int(is_q ? hg : hg - P.q_groups) * kRows;
  const int n = min(kRows, (is_q ? P.hq : P.hkv) - h0);
  const int b = P.batch == 1 ? 0 : int(row / uint32_t(P.tokens)), t = int(row - uint32_t(b) * uint32_t(P.tokens));

  Pack4<T> raw[kRows][2];
  const T* in = static_cast<const T*>(S.in) + b * S.in_b + t * S.in_t + h0 * S.in_h + 4 * lane;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (r < n) {
      raw[r][0].v = load_row<kRows>(in + r * S.in_h);
      raw[r][1].v = load_row<kRows>(in + r * S.in_h + 64);
    }
  }
  // The row of the angle table; a position outside the table gives NaN rows.
  int64_t pos = t + int64_t(b) * P.table_b_rows;
  if (P.positions) {
    const int64_t i = b * P.pos_b + t * P.pos_t;
    pos = P.pos64 ? static_cast<const int64_t*>(P.positions)[i] : static_cast<const int32_t*>(P.positions)[i];
  }
  const bool known = pos >= 0 && pos < P.table_rows;
  // c[i], s[i]: rotation of pair i of this lane (pairs of four channels apart by 64, or adjacent).
  float c[4], s[4];
  if (known) {
    const int64_t base = pos * P.table_stride;
    if (kInterleaved) {
      load_small<2>(P.cos, base + 2 * lane, P.table_dtype, P.table_words, c);
      load_small<2>(P.cos, base + 32 + 2 * lane, P.table_dtype, P.table_words, c + 2);
      load_small<2>(P.sin, base + 2 * lane, P.table_dtype, P.table_words, s);
      load_small<2>(P.sin, base + 32 + 2 * lane, P.table_dtype, P.table_words, s + 2);
    } else {
      load_small<4>(P.cos, base + 4 * lane, P.table_dtype, P.table_words, c);
      load_small<4>(P.sin, base + 4 * lane, P.table_dtype, P.table_words, s);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
  }
  float wl[4] = {1.f, 1.f, 1.f, 1.f}, wh[4] = {1.f, 1.f, 1.f, 1.f};
  if (S.weight) {
    load_small<4>(S.weight, 4 * lane, P.weight_dtype, P.weight_words, wl);
    load_small<4>(S.weight, 64 + 4 * lane, P.weight_dtype, P.weight_words, wh);
  }
  // Pair i of the lane: channels (lo[i], hi[i]), or with adjacent pairs (lo[2i], lo[2i + 1]), then of hi.
  auto first_of = [](const float* lo, const float* hi, int i) {
    return kInterleaved ? (i < 2 ? lo[2 * i] : hi[2 * i - 4]) : lo[i];
  };
  auto second_of = [](const float* lo, const float* hi, int i) {
    return kInterleaved ? (i < 2 ? lo[2 * i + 1] : hi[2 * i - 3]) : hi[i];
  };
  // With x the channels as they are, out_a = inv (x_a ac - x_b bs) and out_b = inv (x_b bc + x_a as), two pairs
  // at a time: the weights are multiplied into the angles once per group instead of once per row.
  uint64_t ac[2], bs[2], bc[2], as[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t c2 = pair_of(c[2 * i], c[2 * i + 1]), s2 = pair_of(s[2 * i], s[2 * i + 1]);
    const uint64_t wa = pair_of(first_of(wl, wh, 2 * i), first_of(wl, wh, 2 * i + 1));
    const uint64_t wb = pair_of(second_of(wl, wh, 2 * i), second_of(wl, wh, 2 * i + 1));
    ac[i] = mul_pair(wa, c2), bc[i] = mul_pair(wb, c2), as[i] = mul_pair(wa, s2);
    bs[i] = mul_pair(wb, pair_of(-s[2 * i], -s[2 * i + 1]));
  }
  float inv[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) inv[r] = 1.0f;
  if (S.weight) {
    float ss[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float x[8];
      raw[r][0].get(x);
      raw[r][1].get(x + 4);
      uint64_t sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint64_t p = pair_of(x[i], x[i + 1]);
        sum = fma_pair(p, p, sum);
      }
      float s0, s1;
      split_pair(sum, s0, s1);
      ss[r] = s0 + s1;
    }
    if constexpr (kRows == 4) {
      // Lanes trade the rows they do not keep: after two steps lane l holds row l / 4, and two more end its sum.
      const bool upper = lane & 8, odd = lane & 4;
      float a = upper ? ss[2] : ss[0], e = upper ? ss[3] : ss[1];
      a += __shfl_xor_sync(group_mask, upper ? ss[0] : ss[2], 8);
      e += __shfl_xor_sync(group_mask, upper ? ss[1] : ss[3], 8);
      float own = odd ? e : a;
      own += __shfl_xor_sync(group_mask, odd ? a : e, 4);
      own += __shfl_xor_sync(group_mask, own, 2);
      own += __shfl_xor_sync(group_mask, own, 1);
      own = rsqrtf(own * (1.0f / kD) + P.eps);
#pragma unroll
      for (int r = 0; r < kRows; ++r) inv[r] = __shfl_sync(group_mask, own, 4 * r, 16);
    } else {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss[0] += __shfl_xor_sync(group_mask, ss[0], o);
      inv[0] = rsqrtf(ss[0] * (1.0f / kD) + P.eps);
    }
  }
  T* out = static_cast<T*>(S.out) + b * S.out_b + t * S.out_t + h0 * S.out_h + 4 * lane;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (r >= n) break;  // uniform in the group
    float lo[4], hi[4], x[4], y[4];  // x, y: the pairs' first and second channels
    raw[r][0].get(lo);
    raw[r][1].get(hi);
    const uint64_t inv2 = pair_of(inv[r], inv[r]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t a = pair_of(first_of(lo, hi, 2 * i), first_of(lo, hi, 2 * i + 1));
      const uint64_t e = pair_of(second_of(lo, hi, 2 * i), second_of(lo, hi, 2 * i + 1));
      split_pair(mul_pair(fma_pair(a, ac[i], mul_pair(e, bs[i])), inv2), x[2 * i], x[2 * i + 1]);
      split_pair(mul_pair(fma_pair(e, bc[i], mul_pair(a, as[i])), inv2), y[2 * i], y[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = kInterleaved ? (i & 1 ? y[i >> 1] : x[i >> 1]) : x[i];
      hi[i] = kInterleaved ? (i & 1 ? y[2 + (i >> 1)] : x[2 + (i >> 1)]) : y[i];
    }
    Pack4<T> p;
    p.set(lo);
    store_row<kRows>(out + r * S.out_h, p);
    p.set(hi);
    store_row<kRows>(out + r * S.out_h + 64, p);
  }
}

// Heads per 16-lane group: four, so that a group has eight loads in flight and reads its angle row
// once for four heads; one where four would leave SMs without a CTA (few rows: latency counts).
constexpr int kRopeRows = 4;

template <typename T>
static void launch_rope(RopeParams& P, cudaStream_t s) {
  const int64_t rows = int64_t(P.batch) * P.tokens;
  P.q_groups = (P.hq + kRopeRows - 1) / kRopeRows;
  P.groups = P.q_groups + (P.hkv + kRopeRows - 1) / kRopeRows;
  const int64_t wide = rows * P.groups;
  if (wide >= 148 * 16) {
    P.n_units = uint32_t(wide);
    const unsigned grid = unsigned((wide + 7) / 8);
    if (P.interleaved) norm_rope_kernel<T, kRopeRows, true><<<grid, 128, 0, s>>>(P);
    else norm_rope_kernel<T, kRopeRows, false><<<grid, 128, 0, s>>>(P);
  } else {
    P.q_groups = P.hq, P.groups = P.hq + P.hkv;
    P.n_units = uint32_t(rows * P.groups);
    const unsigned grid = (P.n_units + 3) / 4;
    if (P.interleaved) norm_rope_kernel<T, 1, true><<<grid, 64, 0, s>>>(P);
    else norm_rope_kernel<T, 1, false><<<grid, 64, 0, s>>>(P);
  }
}

// Rows on boundaries of four elements, as the kernel's words need.
static int check_rows(const void* p, const int64_t* strides, const tp_rope_layout& L, int heads, const char* what) {
  const int bytes = L.dtype == TP_F32 ? 16 : 8;
  if (!p) return fail(TP_ERR_INVALID, std::string("tp_norm_rope: NULL ") + what);
  const bool odd = (L.batch > 1 && strides[0] % 4) || (L.tokens > 1 && strides[1] % 4) || (heads > 1 && strides[2] % 4);
  if (uintptr_t(p) % bytes || odd)
    return fail(TP_ERR_INVALID, std::string("tp_norm_rope: rows of ") + what + " must start on boundaries of 4 elements");
  return TP_OK;
}

static RopeSide rope_side(const void* in, void* out, const void* weight, const int64_t* si, const int64_t* so) {
  return RopeSide{in, out, weight, si[0], si[1], si[2], so[0], so[1], so[2]};
}

}  // namespace tp

using namespace tp;

extern "C" int tp_norm_rope(const tp_rope_layout* layout, const void* q, const void* k, const void* q_weight,
                            const void* k_weight, const void* cos, const void* sin, const void* positions, void* q_out,
                            void* k_out, void* stream) {
  if (!layout) return fail(TP_ERR_INVALID, "tp_norm_rope: NULL layout");
  const tp_rope_layout& L = *layout;
  auto known = [](int d) { return d == TP_F16 || d == TP_F32 || d == TP_BF16; };
  if (!known(L.dtype) || !known(L.weight_dtype) || !known(L.table_dtype))
    return fail(TP_ERR_INVALID, "tp_norm_rope: dtype must be float16, bfloat16 or float32");
  if (L.batch < 0 || L.tokens < 0) return fail(TP_ERR_INVALID, "tp_norm_rope: negative size");
  if (L.q_heads < 1 || L.k_heads < 1)
    return fail(TP_ERR_INVALID, "tp_norm_rope: q and k need at least one head each");
  if (L.batch == 0 || L.tokens == 0) return TP_OK;
  int st = check_rows(q, L.q_in, L, L.q_heads, "q");
  if (st == TP_OK) st = check_rows(k, L.k_in, L, L.k_heads, "k");
  if (st == TP_OK) st = check_rows(q_out, L.q_out, L, L.q_heads, "q_out");
  if (st == TP_OK) st = check_rows(k_out, L.k_out, L, L.k_heads, "k_out");
  if (st != TP_OK) return st;
  if (!cos || !sin) return fail(TP_ERR_INVALID, "tp_norm_rope: NULL angle table");
  if (L.table_rows < 0 || (L.table_rows > 1 && L.row_stride < 64))
    return fail(TP_ERR_INVALID, "tp_norm_rope: angle rows must be at least 64 elements apart");
  if (!positions && int64_t(L.batch_rows) * (L.batch - 1) + L.tokens > L.table_rows)
    return fail(TP_ERR_INVALID, "tp_norm_rope: the angle table has fewer rows than tokens");
  const int64_t heads = int64_t(L.q_heads) + L.k_heads, tokens = int64_t(L.batch) * L.tokens;
  if (heads > (1 << 20) || tokens > (int64_t(1) << 31) / heads)
    return fail(TP_ERR_INVALID, "tp_norm_rope: more than 2^31 rows");
  RopeParams P;
  P.q = rope_side(q, q_out, q_weight, L.q_in, L.q_out);
  P.k = rope_side(k, k_out, k_weight, L.k_in, L.k_out);
  P.cos = cos;
  P.sin = sin;
  P.positions = positions;
  P.table_stride = L.row_stride;
  P.pos_b = L.pos_strides[0];
  P.pos_t = L.pos_strides[1];
  P.batch = L.batch;
  P.tokens = L.tokens;
  P.hq = L.q_heads;
  P.hkv = L.k_heads;
  P.table_rows = L.table_rows;
  P.table_b_rows = L.batch_rows;
  P.pos64 = L.pos64;
  P.table_dtype = L.table_dtype;
  P.weight_dtype = L.weight_dtype;
  P.interleaved = L.interleaved;
  P.eps = L.eps;
  const int tw = L.table_dtype == TP_F32 ? 16 : 8, ww = L.weight_dtype == TP_F32 ? 16 : 8;
  P.table_words = (uintptr_t(cos) | uintptr_t(sin)) % tw == 0 && (L.row_stride % 4 == 0 || L.table_rows == 1);
  P.weight_words = (uintptr_t(q_weight) | uintptr_t(k_weight)) % ww == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L.dtype == TP_F16) launch_rope<__half>(P, s);
  else if (L.dtype == TP_BF16) launch_rope<__nv_bfloat16>(P, s);
  else launch_rope<float>(P, s);
  return check_launch("tp_norm_rope");
}
