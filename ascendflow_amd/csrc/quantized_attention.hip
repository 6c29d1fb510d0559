// Attention of grouped query heads over a paged cache held in 8 bits, for gfx950.
//
// A block of GROUP tokens of a key/value head has a key scale a and a value scale b; its
// codes k, v stand for a k and b v. For query row q (a token's head) over the keys j it sees
//   s_j = scale a_j (q . k_j),  out = sum_j e^s_j b_j v_j / sum_j e^s_j.
// Codes of either kind are exact in the query's 16-bit type, so both products run on the
// 16-bit matrix instructions with codes converted on the way and scales kept out of them:
// x_j = s_j log2(e) + log2 b_j is the exponent of a weight in units of its values' scale,
//   p_j = 2^(x_j - m),  out = sum_j p_j v_j / sum_j p_j / b_j,  m the running maximum of x.
// So the scales cost one multiply-add per 16 keys instead of one per element, and the
// weight that contributes most is 1, which no type rounds. Scales count as at least 2^-80
// (append writes none below), so that 1 / b is a number. Their ratios are not bounded by
// that (append writes up to 2^122): a p_j of 0 may stand for a key that counts in the
// denominator. Where the value scales of a tile's keys lie that far apart, the wave sums
// its denominators anew (sum_weights).
//
// The sums, the maximum and the output are float32; p is rounded to the query's type (a
// matrix operand has to be), at most half a step of each weight, while the denominator
// sums the weights before rounding. float16 raises the maximum only when it grows by more
// than 2^8, bfloat16, whose step is coarser, whenever it grows.
#include <algorithm>
#include <cmath>
#include <utility>

#include "shares.h"
#include "../../include/ascendflow_amd.h"

namespace afa {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT> __device__ constexpr float q8_tau() { return DT == DT_F16 ? 8.0f : 0.0f; }
constexpr float Q8_LEAST_SCALE = 8.271806125530277e-25f;  // 2^-80

// The larger of v and a positive bound; compared by bits, so that a NaN stays one.
__device__ __forceinline__ float at_least(float v, float bound) {
  return __int_as_float(max(__float_as_int(v), __float_as_int(bound)));
}

// A row's running maximum before its first key. Finite, and below every score of a key.
constexpr float Q8_NO_MAXIMUM = -3.402823466e+38f;

// Weights are 2^(s sk + (lv - m)) with one rounding, of a maximum m = s sk + lv that was rounded: what that rounding
// took is a factor of every weight of a row, at most 2 up to |m| = 2^24. From there on it could leave the range: s sk + lv
// takes the place of s then, rounded as m is, with 1 for sk and 0 for lv.
constexpr float Q8_FAR = 16777216.0f;  // 2^24
__device__ __forceinline__ bool q8_far(float m) {  // there is a maximum, finite and far from zero
  return (__float_as_uint(m) & 0x7fffffffu) - __float_as_uint(Q8_FAR) < __float_as_uint(-Q8_NO_MAXIMUM) - __float_as_uint(Q8_FAR);
}

// Whether sums of p_j / b_j over that many keys may lack some that count, given the least and the most of their value scales.
// p is 0 below 2^-126, rescaling drops no more than that, and m is at most the largest weight's exponent + log2 of the largest b
// (bfloat16; float16's may be 2^8 less than it will be): what is dropped of a key is under 2^(spread - 126) of the largest
// weight, of all keys under 2^-26.
template <int DT>
__device__ __forceinline__ bool far_apart(float least, float most, int keys) {
  const int spread = (uniform(__float_as_int(most)) >> 23) - (uniform(__float_as_int(least)) >> 23) + 1;
  return spread + (32 - __clz(keys)) > 100 - (int)q8_tau<DT>();
}

// v 2^e for a result inside float32's range, subnormal ones included.
__device__ __forceinline__ float times_exp2(float v, float e) {
  const bool low = e < 0.f;
  return v * fast_exp2(e + (low ? 64.f : -64.f)) * (low ? 5.42101086e-20f : 1.84467441e+19f);
}

// Denominators total_p of parts whose maxima are m_p, as of one part whose maximum is `top`: sum_p 2^(m_p - top) total_p.
// The weights may be 0 where the products are not, so a part's exponent goes into the weight's, in units of 2^unit, the
// largest of the products' exponents.
__device__ __forceinline__ float part_exponent(float m, float total, float top) {
  return (m - top) + (float)__builtin_amdgcn_frexp_expf(total);
}
__device__ __forceinline__ float part_weight(float m, float total, float top, float unit) {
  return __builtin_amdgcn_frexp_mantf(total) * fast_exp2(part_exponent(m, total, top) - unit);
}
// Whether the plain sum lacks a product: a weight that is 0 next to a total that is not.
__device__ __forceinline__ bool weight_lost(float m, float total, float top) { return m - top < -126.f && total > 0.f; }

// ln(sum of e^scores), also of a denominator below float32's normal numbers.
__device__ __forceinline__ float q8_lse(float m, float total) {
  const bool low = __float_as_uint(total) - 1u < 0x007fffffu;
  return row_lse(low ? m - 64.f : m, low ? total * 1.84467441e+19f : total);
}

struct QuantizedArgs {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  const int32_t* cu;
  const int32_t* used;
  void* out;
  float* lse;  // [T][HKV * H] or NULL
  int64_t q_t, q_h, o_t, o_h;
  int32_t T, B, HKV, W, page_shift, group_shift, blocks, causal;
  int32_t H;  // query heads of a key/value head: the packed rows of a token
  float scale;
  int32_t workers;          // workgroups of the same key/value heads
  float* partial_o;         // [2 * workers][HKV][ROWS / 16][D / 16][64][4], not normalised, as a wave holds it
  float* partial_ml;        // [2 * workers][HKV][ROWS][2]: running maximum (log2), sum of weights
  TileRecord* records;      // [tiles], alike for every head
  uint32_t* tile_count;
  uint32_t tiles;
};

// ---- codes ---------------------------------------------------------------------

// Eight codes (the bytes of lo, then of hi) as a matrix operand.
template <int DT, int CT> struct Codes;
template <> struct Codes<DT_BF16, AFA_CODE_E4M3> {
  static __device__ __forceinline__ bf16x8 decode(uint32_t lo, uint32_t hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};
template <> struct Codes<DT_F16, AFA_CODE_E4M3> {
  static __device__ __forceinline__ f16x8 decode(uint32_t lo, uint32_t hi) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    typedef uint32_t one;
    const u32x4 w = {__builtin_bit_cast(one, a), __builtin_bit_cast(one, b), __builtin_bit_cast(one, c),
                     __builtin_bit_cast(one, d)};
    return __builtin_bit_cast(f16x8, w);
  }
};
// int8 to float16: with its sign bit turned a byte is c + 128, behind the exponent of 2^10
// it reads 1024 + 128 + c, exactly.
template <> struct Codes<DT_F16, AFA_CODE_INT8> {
  static __device__ __forceinline__ f16x8 decode(uint32_t lo, uint32_t hi) {
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    auto two = [&](uint32_t bytes, uint32_t select) {
      const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, bytes, select)) - bias;
      return __builtin_bit_cast(uint32_t, h);
    };
    const u32x4 w = {two(lo, 0x07010700u), two(lo, 0x07030702u), two(hi, 0x07010700u), two(hi, 0x07030702u)};
    return __builtin_bit_cast(f16x8, w);
  }
};
// int8 to bfloat16: eight significant bits hold every code, so the upper half of its float32 is all of it.
template <> struct Codes<DT_BF16, AFA_CODE_INT8> {
  static __device__ __forceinline__ bf16x8 decode(uint32_t lo, uint32_t hi) {
    auto two = [&](uint32_t bytes, int at) {
      const float a = (float)(int8_t)(bytes >> at), b = (float)(int8_t)(bytes >> (at + 8));
      return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    };
    const u32x4 w = {two(lo, 0), two(lo, 16), two(hi, 0), two(hi, 16)};
    return __builtin_bit_cast(bf16x8, w);
  }
};

// ---- denominators anew ---------------------------------------------------------

// total = sum_j 2^(x_j - m - log2 b_j) over a wave's keys, each weight an exponential of its own next to a maximum of
// their own, so that none is lost however far the value scales lie apart; x_j and m as the numerators have them. It reads
// the keys once more, straight from the cache: the price of scales that far apart (64 requests of 16K 283 -> 564 us, 2000
// tokens behind 18K 618 -> 2134). The range of the scales and the joins that tell cost other calls up to 2% (one request of
// 4K 20.6 -> 20.9 us, 48 x 4 tokens 38.5 -> 39.2 in a graph).
// Operand f of lane group g's queries holds columns column(f, g) .. + 7; group i is the 16 keys from first_key(i) on.
template <int DT, int CT, int D, int QT, typename X8, typename Column, typename Key>
__device__ __forceinline__ void sum_weights(const QuantizedArgs& a, const int32_t* table, int kv_head, int kv_end,
                                            float scale_log2, int groups, Key&& first_key, Column&& column,
                                            const X8 (&qf)[QT][D / 32], const int (&limit)[QT], const float (&m)[QT],
                                            float (&total)[QT]) {
  const int lane = (int)opaque(threadIdx.x) & 63, g = lane >> 4, i16 = lane & 15;  // worked out here, not ahead of the loops
  float top[QT], sum[QT];
  bool far[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    top[qt] = Q8_NO_MAXIMUM;
    sum[qt] = 0.f;
    far[qt] = q8_far(m[qt]);
  }
#pragma unroll 1
  for (int i = 0; i < groups; ++i) {
    const int key = uniform(first_key(i));
    if (key >= kv_end) continue;
    const int id = uniform(table[min(key >> a.page_shift, a.W - 1)]);
    if ((uint32_t)id >= (uint32_t)a.blocks) continue;
    const int64_t row = ((int64_t)id << a.page_shift) + (key & ((1 << a.page_shift) - 1));
    const int64_t block = (row >> a.group_shift) * a.HKV + kv_head;
    const float sk = at_least(a.k_scale[block] * scale_log2, 1.17549435e-38f);
    const float lv = __log2f(at_least(a.v_scale[block], Q8_LEAST_SCALE));
    const uint8_t* const codes = a.k + ((row + i16) * a.HKV + kv_head) * D;
    f32x4 s[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) s[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < D / 32; ++f) {
      const u32x2 w = *(const u32x2*)(codes + column(f, g));
      const X8 kf = Codes<DT, CT>::decode(w[0], w[1]);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[qt] = B16<DT>::mfma(kf, qf[qt][f], s[qt]);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float e[4], most = -INFINITY;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float near = __builtin_fmaf(s[qt][r], sk, lv - m[qt]), away = __builtin_fmaf(s[qt][r], sk, lv) - m[qt];
        e[r] = key + 4 * g + r < limit[qt] ? (far[qt] ? away : near) - lv : -INFINITY;
        most = fmaxf(most, e[r]);
      }
      const float now = fmaxf(top[qt], max_over_lane_groups(most));
      sum[qt] *= fast_exp2(top[qt] - now);
      top[qt] = now;
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[qt] += fast_exp2(e[r] - now);
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float all = times_exp2(sum_over_lane_groups(sum[qt]), fmaxf(top[qt], -200.f));
    // A sum that is not a number stays so.
    total[qt] = (__float_as_uint(total[qt]) & 0x7fffffffu) > 0x7f800000u ? total[qt] : all;
  }
}

// ---- stream form ---------------------------------------------------------------
//
// For the few rows of decode and verification: a tile is 16 QT packed rows of one
// key/value head. A workgroup's four waves take HW heads, whose rows of a token lie side
// by side in memory, and 4 / HW runs of 32 cache rows of a chunk. Waves are on their own
// until a tile ends: each keeps all rows' queries, an output of its own and a ring of LDS
// slots that the load-to-LDS path fills ahead of their use, without a barrier or a
// register; it waits for its own loads only.
// S^T[keys, rows] = K Q^T: a lane reads 16 bytes of a key row (the order of columns is
// free, queries follow it). O^T[columns, rows] += V^T P^T: the accumulator layout of S^T
// is the operand layout of P^T, and ds_read_b64_tr_b8 gives a lane a column's codes of the
// eight keys whose weights it holds. Codes become 16-bit values between LDS and the
// matrix instructions. Bound by HBM where requests are many or long (64 of 8K to 16K, 8
// heads of 128 columns 280 us, 6.1 TB/s; 342 with rows kept in registers a chunk ahead and a
// head a workgroup), by a cold start and the join where they are few (one of 4K 13 us). 32
// rows of 256 columns, or of one head of 128, spill 10 to 38 registers, around the chunk loop.
template <int QT, int HW> struct StreamForm {
  static constexpr int ROWS = 16 * QT, KEYS = 128 / HW, THREADS = 256;
  static constexpr uint32_t START = 1, LEAST = 2;
  static constexpr float JOIN = 4.0f;
};
// Slots of a wave's ring, 64 D bytes each, for two workgroups per CU (D = 256: one).
template <int D> __host__ __device__ constexpr int q8_slots() { return D == 64 ? 4 : 2; }
template <int D> __host__ __device__ constexpr int q8_groups() { return D == 256 ? 1 : 2; }  // workgroups of a CU

template <int BYTES> struct Bytes;
template <> struct Bytes<8> { typedef u32x2 type; };
template <> struct Bytes<16> { typedef u32x4 type; };

// Unit u (16 bytes) of row r of a slot's keys lies at u ^ key_swizzle(r): in a 16-byte read
// the rows {0..3, 12..15} take unit u and {4..11} unit u ^ 1 at once (or the other way
// round), which then fall on 16 distinct 16-byte groups of LDS's 256 bytes.
template <int D> __device__ __forceinline__ int key_swizzle(int r) {
  return D == 64 ? (-(r >> 2)) & 3 : D == 128 ? (r >> 1) & 7 : r & 15;
}
// The same for values: a half of a transposing read takes unit u of rows 0..7 (or 8..15)
// and of the 16 rows further.
template <int D> __device__ __forceinline__ int value_swizzle(int r) {
  const int t = r >> 4;
  return D == 64 ? ((r >> 2) & 1) | (t << 1) : D == 128 ? ((r >> 1) & 3) | (t << 2) : (r & 7) | (t << 3);
}

// Waits until at most n <= MOST slots' loads (PER each) are in flight.
template <int PER, int MOST>
__device__ __forceinline__ void wait_slots(int n) {
  static_assert(PER * MOST < 64, "vmcnt holds 6 bits");
  if constexpr (MOST > 0) {
    if (n < MOST) {
      wait_slots<PER, MOST - 1>(n);
      return;
    }
  }
  wait_vmcnt<PER * MOST>();
}

// STREAM: non-temporal loads, for requests of one tile each (nothing is read twice but
// pages that requests share, a case not measured) over caches too large to stay in the
// 256 MiB Infinity Cache, rows of whole 128-byte lines.
template <int DT, int CT, int D, int QT, int HW, bool STREAM>
__global__ __launch_bounds__(256, q8_groups<D>()) void quantized_stream_kernel(QuantizedArgs a) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x8 x8;
  typedef typename B16<DT>::x4 x4;
  typedef StreamForm<QT, HW> F;
  constexpr int ROWS = F::ROWS, KEYS = F::KEYS, KW = 4 / HW, KL = D / 64, VT = D / 16;
  constexpr int NS = q8_slots<D>(), V_AT = 32 * D, META_AT = 64 * D, SLOT = META_AT + 256;
  constexpr int LOADS = 32 * D / 1024, LR = 1024 / D;  // of keys or values; rows of a load
  constexpr int ALL_LOADS = 2 * LOADS + 1;
  // Eight float32 numbers stand between eight int8 codes and bfloat16: converted where they are used, since the compiler
  // would have those of many fragments at once and spill up to 362 registers (64 requests of 8K, 8 heads of 128 columns
  // 222 us instead of 185, 32 x 4 tokens of 64 heads of 256 columns behind 4000 427 instead of 129).
  auto values_of = [](uint32_t lo, uint32_t hi) {
    if constexpr (DT == DT_BF16 && CT == AFA_CODE_INT8) __asm__ volatile("" : "+v"(lo), "+v"(hi));
    return Codes<DT, CT>::decode(lo, hi);
  };
  __shared__ __attribute__((aligned(256))) uint8_t ring[4][NS][SLOT];
  __shared__ float2 joined_ml[4][QT][16];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, i16 = lane & 15;
  const int H = a.H;
  // Heads of one worker side by side on one XCD: together they read whole rows.
  const uint32_t index = xcd_contiguous(blockIdx.x, gridDim.x), groups = (uint32_t)a.HKV / HW;
  const int kv_head = uniform((int)(index % groups) * HW + wave % HW);
  const int part = wave / HW;  // this wave's run of a chunk's rows
  const uint32_t worker = (uint32_t)uniform((int)(index / groups));

  TileShare share;
  if (!find_share<F>(a, worker, worker, share)) return;
  int request = share.request;
  uint32_t place = share.place, offset = share.offset;
  uint64_t left = share.end - share.begin;
  const float scale_log2 = a.scale * LOG2E;
  const uint32_t row_bytes = (uint32_t)a.HKV * D;
  const uint32_t ring_base = lds_address(ring[0]) + (uint32_t)wave * (NS * SLOT);

  // Load p of a slot's keys or values brings rows LR p .. + LR - 1 of it, 16 bytes a lane.
  const int ln_row = lane / (D / 16), ln_unit = lane % (D / 16);
  auto load16 = [](uint32_t to, uint32_t off, const uint8_t* from) {
    if constexpr (STREAM)
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" :: "s"(to), "v"(off), "s"(from) : "memory");
    else
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(off), "s"(from) : "memory");
  };
  // Fragment addresses inside a slot; the XOR of a column group picks its unit.
  const int rv = 16 * (i16 >> 3) + 4 * g + ((i16 >> 1) & 3);
  const uint32_t k_at = (uint32_t)(i16 * D + ((g ^ key_swizzle<D>(i16)) << 4));
  const uint32_t v_at = (uint32_t)(V_AT + rv * D + (value_swizzle<D>(rv) << 4) + (i16 & 1) * 8);

  for (bool first_part = true;; first_part = false) {
    if (request >= a.B) return;  // never, unless cu_seqlens_q or seqused_kv change under the call
    const TileSpan<F, QuantizedArgs> span(a, request);
    if (place >= span.tiles) {  // on to the next request that has tokens (there is one: something is left)
      share.tiles_before += span.tiles;
      place = 0;
      ++request;
      continue;
    }
    const uint32_t tile = (uint32_t)uniform((int)span.tile(place));
    const uint32_t each = (uint32_t)uniform((int)span.counts(place));
    if (share.apart && offset > 0) {  // an earlier workgroup's tile
      if (left <= each - offset) return;
      left -= each - offset;
      offset = 0;
      ++place;
      continue;
    }
    int start, count;
    request_tokens(constant(a.cu), request, a.T, start, count);
    int used, ahead;
    request_rows(a, request, start, used, ahead);
    const int rows = count * H;
    auto visible = [&](int t) { return a.causal ? min(max(ahead + t + 1, 0), used) : used; };
    const int kv_end = visible((min((int)(tile + 1) * ROWS, rows) - 1) / H);
    const int clean_end = visible((int)tile * ROWS / H);  // no row of the tile hides a key below
    const int all_chunks = (kv_end + KEYS - 1) / KEYS;
    const uint32_t stop = share.apart ? each : (uint32_t)min((uint64_t)each, (uint64_t)offset + left);
    auto cut = [&](uint32_t x) {
      return x >= each ? all_chunks : (x <= F::START ? 0 : (int)((uint64_t)(x - F::START) * (uint32_t)all_chunks / (each - F::START)));
    };
    const int begin = cut(offset), chunks = cut(stop);
    const bool whole = offset == 0 && stop == each;
    if (!share.apart && offset == 0 && tid == 0 && index % groups == 0 && share.tiles_before + place < a.tiles) {
      const uint64_t tile_end = share.end - left + each;  // in the sequence
      TileRecord r;
      r.start = start;
      r.row = (int)tile * ROWS;
      r.rows = min(ROWS, rows - (int)tile * ROWS);
      r.first = (int)worker;
      r.last = (int)((tile_end * (uint32_t)share.workers - 1) / share.total);
      a.records[share.tiles_before + place] = r;
    }
    left -= min(left, (uint64_t)(stop - offset));

    // ---- cache rows to LDS: slot (chunk - begin) % NS holds this wave's 32 rows of a chunk ----
    const int32_t* const table = a.table + (int64_t)request * a.W;
    const int page_mask = (1 << a.page_shift) - 1;
    // Chunks of which this wave has rows.
    const int mine = min(chunks, (kv_end - part * 32 + KEYS - 1) / KEYS);
    struct Pages { int id[2]; };  // of the two groups of 16 rows
    auto key_of = [&](int chunk, int t) { return chunk * KEYS + part * 32 + 16 * t; };
    auto holds = [&](const Pages& p, int chunk, int t) {
      return key_of(chunk, t) < kv_end && (uint32_t)p.id[t] < (uint32_t)a.blocks;
    };
    auto slot_of = [&](int chunk) { return ring_base + (uint32_t)((chunk - begin) % NS) * SLOT; };
    // Rows that are not there read the cache's first ones instead (hidden later).
    auto cache_row = [&](const Pages& p, int chunk, int t) -> int64_t {
      return holds(p, chunk, t) ? ((int64_t)p.id[t] << a.page_shift) + (key_of(chunk, t) & page_mask) : 0;
    };
    // A slot comes with 64 words: scales of its two groups' keys (words 0, 1) and values (2, 3), page numbers of the
    // wave's rows NS chunks on (4, 5) and its own (6, 7). All that a step needs is in LDS before it: a scalar load
    // that misses would hold up every LDS read behind it.
    const int role = lane & 7;
    auto fetch = [&](const Pages& p, int chunk) {
      const uint32_t slot = slot_of(chunk);
      const int64_t row[2] = {cache_row(p, chunk, 0), cache_row(p, chunk, 1)};
      const int64_t block = ((role & 1 ? row[1] : row[0]) >> a.group_shift) * a.HKV + kv_head;
      const int entry = key_of(chunk + (role < 6 ? NS : 0), role & 1) >> a.page_shift;
      const void* from = role < 2 ? (const void*)(a.k_scale + block)
                         : role < 4 ? (const void*)(a.v_scale + block) : (const void*)(table + min(entry, a.W - 1));
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                       :: "s"(opaque_uniform(slot + META_AT)), "v"(from) : "memory");
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
          const int t = l / (LOADS / 2), r = l * LR + ln_row;
          const int unit = ln_unit ^ (which ? value_swizzle<D>(r) : key_swizzle<D>(r & 15));
          load16(opaque_uniform(slot + (uint32_t)(which * V_AT + l * 1024)), (uint32_t)(r & 15) * row_bytes + ((uint32_t)unit << 4),
                 (which ? a.v : a.k) + (row[t] * row_bytes + kv_head * D));
        }
    };

    if (KW > 1 && !first_part) __syncthreads();  // the ring's other use is over
    Pages first[NS];  // page numbers of the first chunks, before any load to LDS: one wait for all
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) first[i].id[t] = constant(table)[min(key_of(begin + i, t) >> a.page_shift, a.W - 1)];

    // Queries: columns 64 l + 16 g + 8 h .. + 7 of row i16 are operand 2 l + h.
    x8 qf[QT][2 * KL];
    int limit[QT];  // keys that this lane's row sees
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int row = (int)tile * ROWS + qt * 16 + i16;
      const bool valid = row < rows;
      const int token = valid ? row / H : 0, head = kv_head * H + (valid ? row - token * H : 0);
      limit[qt] = valid ? visible(token) : 0;
      const scalar* q = (const scalar*)a.q + (int64_t)(start + token) * a.q_t + (int64_t)head * a.q_h + 16 * g;
#pragma unroll
      for (int l = 0; l < KL; ++l)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          qf[qt][2 * l + h] = valid ? *(const x8*)(q + 64 * l + 8 * h) : __builtin_bit_cast(x8, u32x4{0u, 0u, 0u, 0u});
    }

    f32x4 o[QT][VT];
    float m_run[QT], l_run[QT];
    float least_scale = INFINITY, most_scale = 0.f;  // of this wave's values (1 where a group has no page)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m_run[qt] = Q8_NO_MAXIMUM;  // finite: a chunk that hides all its keys gives p = 0, never NaN
      l_run[qt] = 0.f;
#pragma unroll
      for (int c = 0; c < VT; ++c) o[qt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (begin + i < mine) {
        fetch(first[i], begin + i);
      }

    // A step's keys and words are in registers before it, read while the step before multiplies its values.
    u32x4 k[2][KL], meta[2];
    auto read_keys = [&](int chunk) {
      const uint32_t slot = slot_of(chunk), base = slot + k_at;
#pragma unroll
      for (int l = 0; l < KL; ++l)
#pragma unroll
        for (int t = 0; t < 2; ++t) k[t][l] = *(const AFA_LDS u32x4*)(lds_at<uint8_t>(base ^ (uint32_t)(l << 6)) + t * 16 * D);
      meta[0] = *lds_at<u32x4>(slot + META_AT);
      meta[1] = *lds_at<u32x4>(slot + META_AT + 16);
    };
    if (begin < mine) {
      wait_slots<ALL_LOADS, NS - 1>(min(NS - 1, mine - 1 - begin));
      __asm__ volatile("" ::: "memory");
      read_keys(begin);
    }
    for (int c = begin; c < mine; ++c) {
      const int key0 = key_of(c, 0);
      const uint32_t slot = slot_of(c);
      const Pages own = {{uniform((int)meta[1][2]), uniform((int)meta[1][3])}}, next = {{uniform((int)meta[1][0]), uniform((int)meta[1][1])}};
      const bool good[2] = {holds(own, c, 0), holds(own, c, 1)};
      const bool edge = key0 + 32 > clean_end || !(good[0] && good[1]);  // uniform
      if (edge) {
        // Values that nobody sees may be codes of no number, which no weight of 0 would hide: half a row a lane.
        const int r = lane >> 1;
        if (!(key0 + r < kv_end && (r < 16 ? good[0] : good[1]))) {
          const uint32_t at = slot + (uint32_t)(V_AT + r * D + (lane & 1) * (D / 2));
#pragma unroll
          for (int i = 0; i < D / 32; ++i) *(AFA_LDS u32x4*)(uintptr_t)(at + 16u * i) = u32x4{0u, 0u, 0u, 0u};
        }
      }
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      i32x2 v[VT];
#pragma unroll
      for (int c2 = 0; c2 < VT; ++c2)
        v[c2] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((i32x2 AFA_LDS*)(uintptr_t)((slot + v_at) ^ (uint32_t)(c2 << 4)));
      f32x4 s[2][QT];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[t][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int l = 0; l < KL; ++l)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const x8 kf = values_of(k[t][l][2 * h], k[t][l][2 * h + 1]);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) s[t][qt] = B16<DT>::mfma(kf, qf[qt][2 * l + h], s[t][qt]);
          }
      float sk[2], lv[2], iv[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        // Without a page the scales are those of other rows.
        const float ks = good[t] ? __uint_as_float(meta[0][t]) : 1.0f;
        const float vs = good[t] ? at_least(__uint_as_float(meta[0][2 + t]), Q8_LEAST_SCALE) : 1.0f;
        sk[t] = at_least(ks * scale_log2, 1.17549435e-38f);  // not 0: times a hidden score
        lv[t] = __log2f(vs);
        iv[t] = 1.0f / vs;
        least_scale = fminf(least_scale, vs);
        most_scale = fmaxf(most_scale, vs);
      }
      if (c + NS < mine) {
        __builtin_amdgcn_s_waitcnt(WAIT_LGKM0);  // the slot is read
        __asm__ volatile("" ::: "memory");
        fetch(next, c + NS);
      }
      if (edge) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              s[t][qt][r] = good[t] && key0 + 16 * t + 4 * g + r < limit[qt] ? s[t][qt][r] : -INFINITY;
      }
      x8 pf[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float most = fmaxf(fmaxf(s[t][qt][0], s[t][qt][1]), fmaxf(s[t][qt][2], s[t][qt][3]));
          top = fmaxf(top, __builtin_fmaf(most, sk[t], lv[t]));
        }
        const float m_new = fmaxf(m_run[qt], max_over_lane_groups(top));
        if (__ballot(m_new > m_run[qt] + q8_tau<DT>()) != 0ull) {
          const float alpha = fast_exp2(m_run[qt] - m_new);
          l_run[qt] *= alpha;
#pragma unroll
          for (int c2 = 0; c2 < VT; ++c2) o[qt][c2] *= alpha;
          m_run[qt] = m_new;
        }
        float factor[2] = {sk[0], sk[1]}, shift[2] = {lv[0] - m_run[qt], lv[1] - m_run[qt]};
        if (__ballot(q8_far(m_new)) != 0ull) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][qt][r] = __builtin_fmaf(s[t][qt][r], sk[t], lv[t]);
            factor[t] = 1.0f;
            shift[t] = -m_run[qt];
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = fast_exp2(__builtin_fmaf(s[t][qt][r], factor[t], shift[t]));
            sum += w;
            pf[qt][4 * t + r] = (scalar)w;
          }
          l_run[qt] = __builtin_fmaf(sum, iv[t], l_run[qt]);
        }
      }
      if (c + 1 < mine) {
        wait_slots<ALL_LOADS, NS - 1>(min(NS - 1, mine - 2 - c));
        __asm__ volatile("" ::: "memory");
        read_keys(c + 1);
      }
#pragma unroll
      for (int c2 = 0; c2 < VT; ++c2) {
        const x8 vf = values_of((uint32_t)v[c2][0], (uint32_t)v[c2][1]);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) o[qt][c2] = B16<DT>::mfma(vf, pf[qt], o[qt][c2]);
      }
    }

    float total[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) total[qt] = sum_over_lane_groups(l_run[qt]);
    if (__builtin_expect(far_apart<DT>(least_scale, most_scale, kv_end), 0))
      sum_weights<DT, CT, D, QT>(a, table, kv_head, kv_end, scale_log2, 2 * (mine - begin),
                                 [&](int i) { return key_of(begin + (i >> 1), i & 1); },
                                 [](int f, int g) { return 64 * (f >> 1) + 16 * g + 8 * (f & 1); }, qf, limit, m_run, total);
    if constexpr (KW > 1) {
      // The first of a head's waves sums up, through the others' rings, 16 rows at a time.
      static_assert(VT * 1024 <= NS * SLOT, "a wave's output fits its ring");
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        if (qt > 0) __syncthreads();  // the last rows are read
        if (part > 0) {
#pragma unroll
          for (int c = 0; c < VT; ++c) *(AFA_LDS f32x4*)(uintptr_t)(ring_base + (uint32_t)(c * 1024 + lane * 16)) = o[qt][c];
          if (g == 0) joined_ml[wave][qt][i16] = make_float2(m_run[qt], total[qt]);
        }
        __syncthreads();
        if (part == 0) {
          float2 ml[KW];
          ml[0] = make_float2(m_run[qt], total[qt]);
          float top = ml[0].x;
#pragma unroll
          for (int w = 1; w < KW; ++w) {
            ml[w] = joined_ml[wave + w * HW][qt][i16];
            top = fmaxf(top, ml[w].x);
          }
          m_run[qt] = top;
          float weight[KW];
          bool lost = false;
          total[qt] = 0.f;
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            weight[w] = fast_exp2(ml[w].x - top);
            total[qt] = __builtin_fmaf(weight[w], ml[w].y, total[qt]);
            lost |= weight_lost(ml[w].x, ml[w].y, top);
          }
          if (__builtin_expect(__ballot(lost) != 0ull, 0)) {
            float unit = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w) unit = fmaxf(unit, part_exponent(ml[w].x, ml[w].y, top));
#pragma unroll
            for (int w = 0; w < KW; ++w) sum += part_weight(ml[w].x, ml[w].y, top, unit);
            total[qt] = times_exp2(sum, unit);
          }
#pragma unroll
          for (int c = 0; c < VT; ++c) o[qt][c] *= weight[0];
#pragma unroll
          for (int w = 1; w < KW; ++w) {
            const uint32_t from = ring_base + (uint32_t)(w * HW * NS * SLOT + lane * 16);
#pragma unroll
            for (int c = 0; c < VT; ++c) o[qt][c] += weight[w] * *lds_at<f32x4>(from + c * 1024);
          }
        }
      }
    }
    if (part == 0) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const int row = (int)tile * ROWS + qt * 16 + i16;
        if (!whole) {
          // As the registers hold it, [column tile][lane] of four columns: whole kilobytes per store.
          const int64_t at = ((2 * (int64_t)worker + (offset == 0 ? 1 : 0)) * a.HKV + kv_head) * QT + qt;
          float* po = a.partial_o + (at * VT * 64 + lane) * 4;
#pragma unroll
          for (int c = 0; c < VT; ++c) *(f32x4*)(po + c * 256) = o[qt][c];
          if (g == 0) *(float2*)(a.partial_ml + (at * 16 + i16) * 2) = make_float2(m_run[qt], total[qt]);
        } else if (row < rows) {
          const float inv = total[qt] > 0.f ? 1.0f / total[qt] : 0.f;
          const int token = row / H, head = kv_head * H + row - token * H;
          scalar* out = (scalar*)a.out + (int64_t)(start + token) * a.o_t + (int64_t)head * a.o_h + 4 * g;
#pragma unroll
          for (int c = 0; c < VT; ++c) {
            x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[qt][c][i] * inv);
            *(x4*)(out + 16 * c) = v;
          }
          if (a.lse && g == 0) a.lse[(int64_t)(start + token) * (a.HKV * H) + head] = q8_lse(m_run[qt], total[qt]);
        }
      }
    }
    if (left == 0) return;
    offset = 0;
    ++place;
  }
}

// ---- tile form -----------------------------------------------------------------
//
// For chunks of prompts: a tile is 16 QT rows for each of eight waves, whose queries and
// outputs stay in registers; chunks of 64 cache rows go through LDS as 16-bit values, so
// that a code is converted once a workgroup and not once a wave. A wave's codes come into
// registers a step before they are converted and stored (keys two chunks ahead of their
// use, values one; two slots each). Page numbers and the scales' three figures a 16-row
// group (of its keys, the values' exponent and reciprocal) are brought for 64 chunks at
// once, so that a step's loads are its codes' alone and each is waited for by count. QK of
// chunk c + 1 is issued ahead of the softmax of chunk c, whose exponentials run in the
// shadow of the matrix instructions of QK (c + 1) and PV (c). 2000 tokens of 32 heads, 8 of
// them key/value heads, behind 18000: 618 us, 1.01 PFLOP/s; bound by the matrix pipes (41%
// busy), every wave's LDS reads of every row and the exponentials; 506 without loading,
// converting and storing codes. 128 columns spill 63 to 95 registers, 256 columns 19 to 26, all
// outside the chunk loop. 8 x 500 tokens of 16 heads, 4 of them key/value heads of 256 columns,
// behind 3500: 297 to 311 us in each pair of types, 0.8 PFLOP/s.
template <int QT> struct TileForm {
  static constexpr int ROWS = 128 * QT, KEYS = 64, THREADS = 512;
  static constexpr uint32_t START = 5, LEAST = 4;
  static constexpr float JOIN = 0.0f;
};

// Unit u (16 bytes) of key row r lies at u ^ this, units of value rows at u ^ twice value_rows<D>(r): the reads'
// 16-byte (keys) and 32-byte (values, 16 columns of 4 rows a lane group) pieces then fall on distinct banks.
template <int D> __device__ __forceinline__ int key_rows(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
template <int D> __device__ __forceinline__ int value_rows(int r) { return D == 64 ? (r >> 1) & 3 : r & 7; }

// step(0), .., step(N - 1), each number known to the compiler: the unroller gives up on loops as long as the ones below with
// 256 columns, and a loop that is left keeps its operands in memory (500 tokens of 8 requests behind 3500 in f16 3017 us).
template <typename Step, int... F>
__device__ __forceinline__ void each_step(Step&& step, std::integer_sequence<int, F...>) {
  (step(std::integral_constant<int, F>{}), ...);
}
template <int N, typename Step>
__device__ __forceinline__ void each_step(Step&& step) {
  each_step(step, std::make_integer_sequence<int, N>{});
}
#define AFA_STEP(n) [&](auto n) __attribute__((always_inline))

template <int DT, int CT, int D, int QT>
__global__ __launch_bounds__(512, 1) void quantized_tile_kernel(QuantizedArgs a) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x8 x8;
  typedef typename B16<DT>::x4 x4;
  typedef TileForm<QT> F;
  constexpr int ROWS = F::ROWS, KC = F::KEYS, KT = KC / 16, KSTEPS = D / 32, VT = D / 16, RB = 2 * D;
  constexpr int CODES = KC * D / F::THREADS;                 // of a thread, of a chunk's keys or values
  constexpr int PIECE = CODES < 16 ? 8 : 16, PIECES = CODES / PIECE;  // bytes of a load, loads
  constexpr int TPR = D / PIECE;                            // threads of a row
  typedef typename Bytes<PIECE>::type piece;
  __shared__ __attribute__((aligned(256))) uint8_t keys[2][KC * RB], values[2][KC * RB];
  constexpr int GROUPS = KC / 16, AHEAD = F::THREADS / 2 / GROUPS;  // chunks whose figures are brought together
  // Of each group of rows: its page, -1 where it holds no keys; its keys' scale, the exponent of its values', one over that.
  __shared__ int32_t page_ids[2][F::THREADS / 2];
  __shared__ __attribute__((aligned(16))) float key_scale[2][F::THREADS / 2], value_exponent[2][F::THREADS / 2], value_inverse[2][F::THREADS / 2];
  __shared__ __attribute__((aligned(16))) float most_scale[2][4];  // the largest of the keys' scales, of each wave that brings them
  // The range of the values' scales that a thread brought: the bits of the largest, and infinity's less those of the least.
  __shared__ uint32_t value_most[F::THREADS / 2], value_rest[F::THREADS / 2];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, i16 = lane & 15;
  const int H = a.H;
  // Heads first: with eight of them an XCD has a head's tiles, which read the same rows.
  const int kv_head = uniform((int)(blockIdx.x % (uint32_t)a.HKV));
  const uint32_t worker = (uint32_t)uniform((int)(blockIdx.x / (uint32_t)a.HKV));
  TileShare share;
  if (!find_share<F>(a, worker, worker, share)) return;
  int request = share.request;
  uint32_t place = share.place, offset = share.offset;
  uint64_t left = share.end - share.begin;
  const float scale_log2 = a.scale * LOG2E;
  const uint32_t row_bytes = (uint32_t)a.HKV * D;
  const int64_t page_bytes = (int64_t)row_bytes << a.page_shift;
  // This thread's pieces: bytes from their group's first row, and places in a slot of keys or values.
  const int piece_row = tid / TPR, piece_column = tid % TPR;
  const uint32_t piece_off = (uint32_t)(piece_row & 15) * row_bytes + (uint32_t)(PIECE * piece_column);
  const bool odd_row = piece_row & 1;
  const uint32_t key_to = (uint32_t)(piece_row * RB + (((piece_column * (PIECE / 8)) ^ key_rows<D>(piece_row)) << 4));
  const uint32_t value_to = (uint32_t)(piece_row * RB + (((piece_column * (PIECE / 8)) ^ (2 * value_rows<D>(piece_row)) ^
                                                          (PIECE == 16 && odd_row ? 1 : 0)) << 4));

  for (bool first_part = true;; first_part = false) {
    if (request >= a.B) return;  // never, unless cu_seqlens_q or seqused_kv change under the call
    const TileSpan<F, QuantizedArgs> span(a, request);
    if (place >= span.tiles) {  // on to the next request that has tokens (there is one: something is left)
      share.tiles_before += span.tiles;
      place = 0;
      ++request;
      continue;
    }
    const uint32_t tile = (uint32_t)uniform((int)span.tile(place));
    const uint32_t each = (uint32_t)uniform((int)span.counts(place));
    if (share.apart && offset > 0) {  // an earlier workgroup's tile
      if (left <= each - offset) return;
      left -= each - offset;
      offset = 0;
      ++place;
      continue;
    }
    int start, count;
    request_tokens(constant(a.cu), request, a.T, start, count);
    int used, ahead;
    request_rows(a, request, start, used, ahead);
    const int rows = count * H;
    auto visible = [&](int t) { return a.causal ? min(max(ahead + t + 1, 0), used) : used; };
    const int kv_end = visible((min((int)(tile + 1) * ROWS, rows) - 1) / H);
    const int clean_chunks = visible((int)tile * ROWS / H) / KC;  // no row of the tile hides a key of these
    const int all_chunks = (kv_end + KC - 1) / KC;
    const uint32_t stop = share.apart ? each : (uint32_t)min((uint64_t)each, (uint64_t)offset + left);
    auto cut = [&](uint32_t x) {
      return x >= each ? all_chunks : (x <= F::START ? 0 : (int)((uint64_t)(x - F::START) * (uint32_t)all_chunks / (each - F::START)));
    };
    const int begin = cut(offset), chunks = cut(stop);
    const bool whole = offset == 0 && stop == each;
    if (!share.apart && offset == 0 && tid == 0 && kv_head == 0 && share.tiles_before + place < a.tiles) {
      const uint64_t tile_end = share.end - left + each;  // in the sequence
      TileRecord r;
      r.start = start;
      r.row = (int)tile * ROWS;
      r.rows = min(ROWS, rows - (int)tile * ROWS);
      r.first = (int)worker;
      r.last = (int)((tile_end * (uint32_t)share.workers - 1) / share.total);
      a.records[share.tiles_before + place] = r;
    }
    left -= min(left, (uint64_t)(stop - offset));

    // ---- codes to registers, as values to LDS -----------------------------------
    const int32_t* const table = a.table + (int64_t)request * a.W;
    const int page_mask = (1 << a.page_shift) - 1;
    // Pages and figures of AHEAD chunks from `chunk` on, a thread a group of keys or of values.
    auto bring = [&](int chunk) {
      const int t = (int)opaque((uint32_t)tid), at = t & (F::THREADS / 2 - 1), buffer = (chunk - begin) / AHEAD & 1;
      const int key = chunk * KC + 16 * at;
      const int id = key < kv_end ? table[min(key >> a.page_shift, a.W - 1)] : -1;
      const bool there = (uint32_t)id < (uint32_t)a.blocks;
      const bool is_value = t >= F::THREADS / 2;
      float scale = 0.f;
      if (there) {
        const int64_t row = ((int64_t)id << a.page_shift) + (key & page_mask);
        scale = (is_value ? a.v_scale : a.k_scale)[(row >> a.group_shift) * a.HKV + kv_head];
      }
      if (is_value) {
        const float vs = at_least(scale, Q8_LEAST_SCALE);
        value_exponent[buffer][at] = there ? __log2f(vs) : -INFINITY;  // a group without keys weighs nothing
        value_inverse[buffer][at] = there ? 1.0f / vs : 0.0f;
        const uint32_t bits = there ? __float_as_uint(vs) : 0u, rest = there ? 0x7f800000u - bits : 0u;
        if (chunk == begin) {
          value_most[at] = bits;
          value_rest[at] = rest;
        } else {  // in place, without a register more: the loop around has none
          __hip_atomic_fetch_max(&value_most[at], bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          __hip_atomic_fetch_max(&value_rest[at], rest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      } else {
        page_ids[buffer][at] = there ? id : -1;
        float most = at_least(scale * scale_log2, 1.17549435e-38f);  // not 0: times a hidden score
        key_scale[buffer][at] = most;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        if (lane == 0) most_scale[buffer][wave] = most;
      }
    };
    auto buffer_of = [&](int chunk) { return (chunk - begin) / AHEAD & 1; };
    auto group_of = [&](int chunk) { return (chunk - begin) % AHEAD * GROUPS; };
    // Piece n of this thread is of row n * (KC / PIECES) + tid / TPR of a chunk, and a wave's are of one group of 16 rows,
    // whose page this is.
    auto piece_group = [&](int n) { return (n * (KC / PIECES) + wave * (64 / TPR)) >> 4; };
    struct Pages { int id[PIECES]; };
    auto pages_of = [&](int chunk) {
      Pages p;
#pragma unroll
      for (int n = 0; n < PIECES; ++n) p.id[n] = uniform(page_ids[buffer_of(chunk)][group_of(chunk) + piece_group(n)]);
      return p;
    };
    typedef const __attribute__((address_space(1))) uint8_t* global_bytes;
    typedef const __attribute__((address_space(1))) piece* global_piece;
    // Every load is made, so that a wait for one counts those behind it: a group without keys reads the cache's first
    // rows, and rows behind the last key are the page's own (hidden when they are stored).
    auto load_codes = [&](const uint8_t* cache, int chunk, const Pages& p, piece (&to)[PIECES]) {
#pragma unroll
      for (int n = 0; n < PIECES; ++n) {
        const int id = p.id[n], key = chunk * KC + 16 * piece_group(n);
        const int64_t at = id >= 0 ? (int64_t)id * page_bytes + (int64_t)(key & page_mask) * row_bytes : 0;
        // In scalar registers, so that a thread's part of the address is one 32-bit register.
        to[n] = *(global_piece)((global_bytes)(uintptr_t)uniform64((uintptr_t)cache + (uint64_t)(at + kv_head * D)) + piece_off);
      }
    };
    auto store_values = [&](const piece (&codes)[PIECES], uint32_t to, bool is_value, int chunk, const Pages& p) {
      to += is_value ? value_to : key_to;
#pragma unroll
      for (int n = 0; n < PIECES; ++n) {
        piece mine = codes[n];
        const int id = p.id[n];
        if (id < 0 || chunk * KC + 16 * piece_group(n) + 16 > kv_end) {
          // Rows that are not there become zeros, which no weight can turn into anything else.
          const int key = chunk * KC + n * (KC / PIECES) + (int)(opaque((uint32_t)tid) / TPR);
          if (id < 0 || key >= kv_end) mine = piece(0);
        }
#pragma unroll
        for (int h = 0; h < PIECE / 8; ++h) {
          uint32_t lo = mine[2 * h], hi = mine[2 * h + 1];
          if (PIECE == 16 && is_value) {  // odd rows the other half first: its turn leaves rows' halves on one another's banks
            lo = odd_row ? mine[2 - 2 * h] : lo;
            hi = odd_row ? mine[3 - 2 * h] : hi;
          }
          __asm__ volatile("" : "+v"(lo), "+v"(hi));  // converted here and not a step ahead, where the registers are taken
          *(AFA_LDS x8*)(uintptr_t)((to ^ (uint32_t)(h << 4)) + (uint32_t)(n * (KC / PIECES) * RB)) = Codes<DT, CT>::decode(lo, hi);
        }
      }
    };

    x8 qf[QT][KSTEPS];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int row = (int)tile * ROWS + (wave * QT + qt) * 16 + i16;
      const bool valid = row < rows;
      const int token = valid ? row / H : 0, head = kv_head * H + (valid ? row - token * H : 0);
      const scalar* q = (const scalar*)a.q + (int64_t)(start + token) * a.q_t + (int64_t)head * a.q_h + 8 * g;
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j)
        qf[qt][j] = valid ? *(const x8*)(q + 32 * j) : __builtin_bit_cast(x8, u32x4{0u, 0u, 0u, 0u});
    }
    // Up to this scale of its keys no score of this wave is far from zero (half of it for lv).
    float far_scale = 0.f;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += fabsf((float)qf[qt][j][e]);
      far_scale = fmaxf(far_scale, sum_over_lane_groups(sum));
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) far_scale = fmaxf(far_scale, __shfl_xor(far_scale, d));
    far_scale = __int_as_float(uniform(__float_as_int(0.5f * Q8_FAR / (far_scale * (CT == AFA_CODE_E4M3 ? 448.0f : 128.0f)))));
    f32x4 o[QT][VT];
    float m_run[QT], l_run[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m_run[qt] = Q8_NO_MAXIMUM;  // finite: a chunk that hides all its keys gives p = 0, never NaN
      l_run[qt] = 0.f;
#pragma unroll
      for (int t = 0; t < VT; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // Fragment addresses (relative to a slot): rows 16 t + i16 of keys, 16 t + 4 g + (i16 >> 2) of values.
    const int rv = 4 * g + (i16 >> 2);
    const uint32_t qk_at = (uint32_t)(i16 * RB + ((g ^ key_rows<D>(i16)) << 4));
    const uint32_t tr_at = (uint32_t)(rv * RB + (value_rows<D>(rv) << 5) + (i16 & 3) * 8);
    constexpr int QK_FRAGS = KSTEPS * KT, LOOK = 5;
    auto qk_chunk = [&](int chunk, f32x4 (&s)[KT][QT], auto&& between) {
      const uint32_t base = opaque(lds_address(keys[chunk & 1]) + qk_at);
      x8 kf[QK_FRAGS];
      auto load = [&](int f) {  // (step j, key tile t)
        const int j = f / KT, t = f % KT;
        kf[f] = *(const AFA_LDS x8*)(lds_at<uint8_t>(base ^ (uint32_t)(j << 6)) + t * 16 * RB);
      };
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[t][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < LOOK; ++f) load(f);
      each_step<QK_FRAGS>(AFA_STEP(step) {
        constexpr int f = decltype(step)::value;
        if constexpr (f + LOOK < QK_FRAGS) load(f + LOOK);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[f % KT][qt] = B16<DT>::mfma(kf[f], qf[qt][f / KT], s[f % KT][qt]);
        between(step);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    constexpr int PV_FRAGS = (KC / 32) * VT;
    auto pv_chunk = [&](int chunk, x8 (&pf)[QT][KC / 32], auto&& between) {
      const uint32_t base = opaque(lds_address(values[chunk & 1]) + tr_at);
      constexpr int VLOOK = 3;
      x4 lo[PV_FRAGS], hi[PV_FRAGS];
      auto load = [&](int f) {  // (32 keys ks, column tile t)
        const int ks = f / VT, t = f % VT;
        const AFA_LDS uint8_t* p = lds_at<uint8_t>(base ^ (uint32_t)((t & 7) << 5)) + (t >> 3) * 256 + ks * 32 * RB;
        lo[f] = B16<DT>::read_tr((const AFA_LDS void*)p);
        hi[f] = B16<DT>::read_tr((const AFA_LDS void*)(p + 16 * RB));
      };
#pragma unroll
      for (int f = 0; f < VLOOK; ++f) load(f);
      each_step<PV_FRAGS>(AFA_STEP(step) {
        constexpr int f = decltype(step)::value, ks = f / VT, t = f % VT;
        if constexpr (f + VLOOK < PV_FRAGS) load(f + VLOOK);
        const x8 vf = {lo[f][0], lo[f][1], lo[f][2], lo[f][3], hi[f][0], hi[f][1], hi[f][2], hi[f][3]};
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) o[qt][t] = B16<DT>::mfma(vf, pf[qt][ks], o[qt][t]);
        between(step);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    auto mask = [&](int chunk, f32x4 (&s)[KT][QT]) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const int row = (int)tile * ROWS + (wave * QT + qt) * 16 + (int)(opaque((uint32_t)tid) & 15u);
        const int lim = visible(min(row, rows - 1) / H) - chunk * KC;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][qt][i] = 16 * t + 4 * g + i < lim ? s[t][qt][i] : -INFINITY;
      }
    };

    auto keys_at = [&](int slot) { return lds_address(keys[0]) + (uint32_t)slot * (KC * RB); };
    auto values_at = [&](int slot) { return lds_address(values[0]) + (uint32_t)slot * (KC * RB); };
    if (!first_part) block_barrier();  // the slots are read
    piece k_codes[PIECES], v_codes[PIECES];
    f32x4 s_a[KT][QT], s_b[KT][QT];
    Pages page1, page2;  // of chunks c + 1 and c + 2 ahead of step c
    if (begin < chunks) {
      bring(begin);
      block_barrier();
      const Pages page0 = pages_of(begin);
      page1 = pages_of(begin + 1);
      page2 = pages_of(begin + 2);
      piece first[PIECES];
      load_codes(a.k, begin, page0, first);
      load_codes(a.v, begin, page0, v_codes);
      load_codes(a.k, begin + 1, page1, k_codes);
      store_values(first, keys_at(begin & 1), false, begin, page0);
      store_values(v_codes, values_at(begin & 1), true, begin, page0);
      load_codes(a.v, begin + 1, page1, v_codes);
      store_values(k_codes, keys_at((begin + 1) & 1), false, begin + 1, page1);
      load_codes(a.k, begin + 2, page2, k_codes);
      block_barrier();
      qk_chunk(begin, s_a, [](auto) {});
    }
    constexpr int HALF = QT * 8, QK_EXP0 = QT + 2, PV_EXP_STEPS = PV_FRAGS / 2 - 1;
    constexpr int STORE_V = 0, STORE_K = QK_FRAGS / 2;  // steps that the stores follow
    int far = 0;  // scores of these chunks may be far from zero
    auto iteration = [&](int c, f32x4 (&cur)[KT][QT], f32x4 (&nxt)[KT][QT]) {
      // Keys of chunk c + 1 and values of c are stored, and every wave is past QK (c) and PV (c - 1),
      // whose slots are free.
      block_barrier();
      const Pages page3 = pages_of(c + 3);
      f32x4 lv;
      float sk[KT], iv[KT];  // scalar registers
      {
        const int buffer = buffer_of(c), at = group_of(c);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          lv[t] = value_exponent[buffer][at + t];
          sk[t] = __int_as_float(uniform(__float_as_int(key_scale[buffer][at + t])));
          iv[t] = __int_as_float(uniform(__float_as_int(value_inverse[buffer][at + t])));
        }
      }
      if (c >= clean_chunks || far) {
        mask(c, cur);
        if (far) {
#pragma unroll
          for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
              for (int i = 0; i < 4; ++i) cur[t][qt][i] = __builtin_fmaf(cur[t][qt][i], sk[t], lv[t]);
            sk[t] = 1.0f;
            lv[t] = 0.0f;
          }
        }
      }
      x8 pf[QT][KC / 32];
      float top[QT], m_new[QT], psum[QT];
      f32x4 shift[QT];
      auto exp_element = [&](int e) {  // (half, qt, key tile of the half, i)
        const int h = e / HALF, qt = (e / 8) % QT, t = 2 * h + (e / 4) % 2, i = e % 4;
        const float p = fast_exp2(__builtin_fmaf(cur[t][qt][i], sk[t], shift[qt][t]));
        psum[qt] = __builtin_fmaf(p, iv[t], psum[qt]);
        pf[qt][h][(t & 1) * 4 + i] = (scalar)p;
      };
      auto qk_between = AFA_STEP(step) {
        constexpr int f = decltype(step)::value;
        if constexpr (f == QK_FRAGS / 2 - 1) __builtin_amdgcn_s_setprio(2);
        if constexpr (f == STORE_V) {
          store_values(v_codes, values_at((c + 1) & 1), true, c + 1, page1);
          load_codes(a.v, c + 2, page2, v_codes);
        }
        if constexpr (f == STORE_K) {
          store_values(k_codes, keys_at(c & 1), false, c + 2, page2);
          load_codes(a.k, c + 3, page3, k_codes);
          page1 = page2;
          page2 = page3;
        }
        if constexpr (f < QT) {
          float m = -INFINITY;
#pragma unroll
          for (int t = 0; t < KT; ++t)
            m = fmaxf(m, __builtin_fmaf(fmaxf(fmaxf(cur[t][f][0], cur[t][f][1]), fmaxf(cur[t][f][2], cur[t][f][3])), sk[t], lv[t]));
          top[f] = m;
        } else if constexpr (f == QT) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            m_new[qt] = fmaxf(m_run[qt], max_over_lane_groups(top[qt]));
            psum[qt] = 0.f;
          }
        } else if constexpr (f == QT + 1) {
          bool grow = false;
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) grow |= m_new[qt] > m_run[qt] + q8_tau<DT>();
          if (__ballot(grow) != 0ull) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              const float alpha = fast_exp2(m_run[qt] - m_new[qt]);
              l_run[qt] *= alpha;
#pragma unroll
              for (int t = 0; t < VT; ++t) o[qt][t] *= alpha;
              m_run[qt] = m_new[qt];
            }
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) shift[qt] = lv - m_run[qt];
        } else {
#pragma unroll
          for (int e = 0; e < HALF; ++e)
            if (QK_EXP0 + e * (QK_FRAGS - QK_EXP0) / HALF == f) exp_element(e);
        }
      };
      auto pv_between = AFA_STEP(step) {
        constexpr int f = decltype(step)::value;
        if constexpr (f == PV_FRAGS / 2 - 1) __builtin_amdgcn_s_setprio(0);
        if constexpr (f < PV_EXP_STEPS) {
#pragma unroll
          for (int e = 0; e < HALF; ++e)
            if (e * PV_EXP_STEPS / HALF == f) exp_element(HALF + e);
        } else if constexpr (f == PV_EXP_STEPS + 1) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) l_run[qt] += psum[qt];
        }
      };
      // Wave priority steps down with the wave's progress through a chunk: of the
      // two waves of a SIMD the one behind wins. The last chunk also runs a QK, over what its slot holds;
      // nobody reads those scores.
      __builtin_amdgcn_s_setprio(3);
      qk_chunk(c + 1, nxt, qk_between);
      __builtin_amdgcn_s_setprio(1);
      pv_chunk(c, pf, pv_between);
    };
    // Step c loads keys of chunk c + 3: the next AHEAD chunks' pages are brought four steps ahead of them, outside of the
    // steps, which then wait for none but their own loads.
    for (int c = begin, until = begin + AHEAD - 4; c < chunks; until += AHEAD) {
      float most = 0.f;
      for (int buffer = 0; buffer < (c == begin ? 1 : 2); ++buffer)
        for (int w = 0; w < 4; ++w) most = fmaxf(most, most_scale[buffer][w]);
      far = uniform(most > far_scale ? 1 : 0);
      for (; c < min(chunks, until); c += 2) {
        iteration(c, s_a, s_b);
        if (c + 1 < chunks) iteration(c + 1, s_b, s_a);
      }
      if (c < chunks) {
        bring(until + 4);
        block_barrier();
      }
    }

    float totals[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) totals[qt] = sum_over_lane_groups(l_run[qt]);
    uint32_t most = 0u, rest = 0u;
    if (begin < chunks) {
#pragma unroll
      for (int i = 0; i < F::THREADS / 2; i += 64) {
        most = max(most, value_most[i + lane]);
        rest = max(rest, value_rest[i + lane]);
      }
    }
    most = (uint32_t)__builtin_amdgcn_readlane((int)wave_max(most), 63);
    rest = (uint32_t)__builtin_amdgcn_readlane((int)wave_max(rest), 63);
    if (__builtin_expect(far_apart<DT>(__uint_as_float(0x7f800000u - rest), __uint_as_float(most), kv_end), 0)) {
      int limit[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) limit[qt] = visible(min((int)tile * ROWS + (wave * QT + qt) * 16 + i16, rows - 1) / H);
      sum_weights<DT, CT, D, QT>(a, table, kv_head, kv_end, scale_log2, (chunks - begin) * GROUPS,
                                 [&](int i) { return begin * KC + 16 * i; }, [](int f, int g) { return 32 * f + 8 * g; }, qf, limit,
                                 m_run, totals);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int group = wave * QT + qt, row = (int)tile * ROWS + group * 16 + i16;
      const float total = totals[qt];
      if (!whole) {
        const int64_t at = ((2 * (int64_t)worker + (offset == 0 ? 1 : 0)) * a.HKV + kv_head) * (ROWS / 16) + group;
        float* po = a.partial_o + (at * VT * 64 + lane) * 4;
        if ((int)tile * ROWS + group * 16 < rows) {
#pragma unroll
          for (int t = 0; t < VT; ++t) *(f32x4*)(po + t * 256) = o[qt][t];
          if (g == 0) *(float2*)(a.partial_ml + (at * 16 + i16) * 2) = make_float2(m_run[qt], total);
        }
      } else if (row < rows) {
        const float inv = total > 0.f ? 1.0f / total : 0.f;
        const int token = row / H, head = kv_head * H + row - token * H;
        scalar* out = (scalar*)a.out + (int64_t)(start + token) * a.o_t + (int64_t)head * a.o_h + 4 * g;
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[qt][t][i] * inv);
          *(x4*)(out + 16 * t) = v;
        }
        if (a.lse && g == 0) a.lse[(int64_t)(start + token) * (a.HKV * H) + head] = q8_lse(m_run[qt], total);
      }
    }
    if (left == 0) return;
    offset = 0;
    ++place;
  }
}

// Combines the parts of the tiles that several workgroups share, in a fixed order:
// out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p. A workgroup takes 16 rows of a head.
// Its waves take a column tile each, and with SPLIT > 1 every SPLIT-th part (few tiles, whose
// parts are many), joined through LDS; AHEAD parts of loads are in flight.
template <int DT, int D, int SPLIT>
__global__ __launch_bounds__(64 * (D / 16) * SPLIT) void quantized_merge_kernel(QuantizedArgs a, int tile_groups) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x4 x4;
  constexpr int VT = D / 16, AHEAD = 4;
  __shared__ f32x4 joined_o[SPLIT > 1 ? SPLIT - 1 : 1][VT][64];
  __shared__ float2 joined_ml[SPLIT > 1 ? SPLIT - 1 : 1][16];
  const uint32_t tile = blockIdx.x / (uint32_t)tile_groups;
  const int group = (int)(blockIdx.x % (uint32_t)tile_groups), kv_head = blockIdx.y;
  if (tile >= *constant((const int32_t*)a.tile_count)) return;
  const TileRecord record = a.records[tile];
  if (record.first == record.last || group * 16 >= record.rows) return;
  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, i16 = lane & 15;
  const int c = wave % VT, sub = wave / VT;
  const int parts = record.last - record.first + 1, mine = (parts - sub + SPLIT - 1) / SPLIT;  // sub, sub + SPLIT, ...
  auto slot = [&](int k) {
    const int p = sub + k * SPLIT;
    return ((2 * (int64_t)(record.first + p) + (p == 0 ? 1 : 0)) * a.HKV + kv_head) * tile_groups + group;
  };
  auto sums = [&](int k) { return *(const float2*)(a.partial_ml + (slot(k) * 16 + i16) * 2); };
  float top = Q8_NO_MAXIMUM, total = 0.f;
#pragma unroll 4
  for (int k = g; k < mine; k += 4) top = fmaxf(top, sums(k).x);
  top = max_over_lane_groups(top);
  bool lost = false;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < mine; k += AHEAD) {
    float2 ml[AHEAD];
    f32x4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int q = min(k + i, mine - 1);
      ml[i] = sums(q);
      v[i] = *(const f32x4*)(a.partial_o + ((slot(q) * VT + c) * 64 + lane) * 4);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float weight = k + i < mine ? fast_exp2(ml[i].x - top) : 0.f;
      total = __builtin_fmaf(weight, ml[i].y, total);
      lost |= weight_lost(ml[i].x, ml[i].y, top);
      o += weight * v[i];
    }
  }
  if (__builtin_expect(__ballot(lost) != 0ull, 0)) {
    float unit = -INFINITY, sum = 0.f;
    for (int k = g; k < mine; k += 4) {
      const float2 ml = sums(k);
      unit = fmaxf(unit, part_exponent(ml.x, ml.y, top));
    }
    unit = max_over_lane_groups(unit);
    for (int k = g; k < mine; k += 4) {
      const float2 ml = sums(k);
      sum += part_weight(ml.x, ml.y, top, unit);
    }
    total = times_exp2(sum_over_lane_groups(sum), unit);
  }
  if constexpr (SPLIT > 1) {
    if (sub > 0) {
      joined_o[sub - 1][c][lane] = o;
      if (c == 0 && g == 0) joined_ml[sub - 1][i16] = make_float2(top, total);
    }
    __syncthreads();
    if (sub > 0) return;
    const float2 own = make_float2(top, total);
#pragma unroll
    for (int w = 0; w < SPLIT - 1; ++w) top = fmaxf(top, joined_ml[w][i16].x);
    lost = weight_lost(own.x, own.y, top);
    const float mine_weight = fast_exp2(own.x - top);
    total *= mine_weight;
    o *= mine_weight;
#pragma unroll
    for (int w = 0; w < SPLIT - 1; ++w) {
      const float2 ml = joined_ml[w][i16];
      const float weight = fast_exp2(ml.x - top);
      total = __builtin_fmaf(weight, ml.y, total);
      lost |= weight_lost(ml.x, ml.y, top);
      o += weight * joined_o[w][c][lane];
    }
    if (__builtin_expect(__ballot(lost) != 0ull, 0)) {
      float unit = part_exponent(own.x, own.y, top);
#pragma unroll
      for (int w = 0; w < SPLIT - 1; ++w) unit = fmaxf(unit, part_exponent(joined_ml[w][i16].x, joined_ml[w][i16].y, top));
      float sum = part_weight(own.x, own.y, top, unit);
#pragma unroll
      for (int w = 0; w < SPLIT - 1; ++w) sum += part_weight(joined_ml[w][i16].x, joined_ml[w][i16].y, top, unit);
      total = times_exp2(sum, unit);
    }
  }
  const int r = group * 16 + i16;
  if (r >= record.rows) return;
  const int packed = record.row + r, token = packed / a.H, head = kv_head * a.H + packed - token * a.H;
  const float inv = total > 0.f ? 1.0f / total : 0.f;
  x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[i] * inv);
  *(x4*)((scalar*)a.out + (int64_t)(record.start + token) * a.o_t + (int64_t)head * a.o_h + 16 * c + 4 * g) = v;
  if (a.lse && c == 0 && g == 0) a.lse[(int64_t)(record.start + token) * (a.HKV * a.H) + head] = q8_lse(top, total);
}

namespace {

bool q8_rows_fit(const void* p, int64_t a, int64_t b) { return ((uintptr_t)p & 15) == 0 && (a | b) % 8 == 0; }

int check_quantized(const QuantizedParams* p) {
  if (!p) return AFA_E_NULL;
  if ((p->dtype != AFA_DTYPE_BF16 && p->dtype != AFA_DTYPE_F16) || (p->code != AFA_CODE_E4M3 && p->code != AFA_CODE_INT8))
    return AFA_E_DTYPE;
  if (p->T < 0 || p->B <= 0 || p->HQ <= 0 || p->HKV <= 0 || p->HQ % p->HKV || p->W <= 0 || p->BLOCKS <= 0) return AFA_E_SHAPE;
  if (p->D != 64 && p->D != 128 && p->D != 256) return AFA_E_SHAPE;
  if (p->GROUP < 16 || (p->GROUP & (p->GROUP - 1)) || p->PAGE < p->GROUP || p->PAGE > (1 << 20) || (p->PAGE & (p->PAGE - 1)))
    return AFA_E_SHAPE;
  // Packed rows, tiles, positions (some chunks past the last too) and the offsets of 16 cache rows are 32-bit numbers.
  if ((int64_t)p->T * p->HQ > 0x7fffff00ll || (int64_t)p->W * p->PAGE > 1ll << 30 || p->B > 0x3fffffff) return AFA_E_SHAPE;
  if (p->HKV > 32768) return AFA_E_SHAPE;
  if (!(p->scale > 0.0f) || !std::isfinite(p->scale)) return AFA_E_SHAPE;
  return AFA_OK;
}

constexpr int Q8_CUS = 256;
constexpr int64_t Q8_STREAM_BYTES = 128ll << 20;

// Form of a call. Tile form (256 rows; D = 256: 128) where a request has more than 256 rows on average and
// its table room for 1536 (2000 tokens of 32 heads, 8 of them key/value heads, behind 18000: 618 us, 924 in the
// stream form with 32 rows; 8 requests of 375 behind 1100 130 and 137; 1 of 1000 behind none 51 and 43, 16 of 48 behind
// 2200 77 and 71). Below, tiles of 32 rows, or 16 where that holds a request. In the stream form a workgroup takes as
// many neighbouring heads as leaves a tile at most 8 workgroups of its own (64 requests of 16K, 8 heads 286 us with 4, 298
// with 2, 336 with 1; one of 16K 58, 39 and 29, since a part a workgroup has to be joined).
struct QuantizedPlan {
  int rows;       // of a tile: 16 or 32 in the stream form, 128 or 256 in the tile form
  int heads;      // key/value heads of a workgroup
  int workers;    // workgroups of such heads
  int64_t tiles;  // the most that monotone cu_seqlens_q can give
  bool stream;    // non-temporal loads
};
QuantizedPlan plan_quantized(const QuantizedParams* p) {
  const int64_t H = p->HQ / p->HKV, each = ((int64_t)p->T + p->B - 1) / p->B * H;  // rows of a request
  QuantizedPlan plan;
  const bool tile_form = each > 256 && (int64_t)p->W * p->PAGE >= 1536;
  plan.rows = tile_form ? (p->D == 256 ? 128 : 256) : each > 16 ? 32 : 16;
  plan.tiles = p->T * H / plan.rows + p->B;
  plan.stream = p->D >= 128 && each <= 16 && 2ll * p->BLOCKS * p->PAGE * p->HKV * p->D >= Q8_STREAM_BYTES;
  plan.heads = tile_form ? 1 : p->HKV % 4 == 0 ? 4 : p->HKV % 2 == 0 ? 2 : 1;
  const int slots = tile_form || p->D == 256 ? Q8_CUS : 2 * Q8_CUS;
  while (plan.heads > 1 && (int64_t)slots * plan.heads / p->HKV > 8 * plan.tiles) plan.heads /= 2;
  plan.workers = std::max(1, slots / (p->HKV / plan.heads));
  return plan;
}
int64_t quantized_part_rows(const QuantizedPlan& plan, int HKV) { return 2ll * plan.workers * HKV * plan.rows; }
uint64_t quantized_bytes(const QuantizedParams* p, const QuantizedPlan& plan) {
  if (p->T == 0) return 0;
  return (uint64_t)(quantized_part_rows(plan, p->HKV) * (p->D + 2) * 4 + plan.tiles * (int64_t)sizeof(TileRecord) + 16);
}

template <int DT, int CT, int D, int QT, int HW>
int launch_stream(const QuantizedArgs& a, const QuantizedPlan& plan, hipStream_t s) {
  const dim3 grid((unsigned)(plan.workers * (a.HKV / HW))), block(256);
  if constexpr (D >= 128 && QT == 1) {
    if (plan.stream) {
      hipLaunchKernelGGL((quantized_stream_kernel<DT, CT, D, QT, HW, true>), grid, block, 0, s, a);
      return (int)hipGetLastError();
    }
  }
  hipLaunchKernelGGL((quantized_stream_kernel<DT, CT, D, QT, HW, false>), grid, block, 0, s, a);
  return (int)hipGetLastError();
}
template <int DT, int CT, int D, int QT>
int launch_heads(const QuantizedArgs& a, const QuantizedPlan& plan, hipStream_t s) {
  if (plan.heads == 4) return launch_stream<DT, CT, D, QT, 4>(a, plan, s);
  if (plan.heads == 2) return launch_stream<DT, CT, D, QT, 2>(a, plan, s);
  return launch_stream<DT, CT, D, QT, 1>(a, plan, s);
}

template <int DT, int CT, int D>
int launch_form(const QuantizedArgs& a, const QuantizedPlan& plan, hipStream_t s) {
  if (plan.rows == 16) return launch_heads<DT, CT, D, 1>(a, plan, s);
  if (plan.rows == 32) return launch_heads<DT, CT, D, 2>(a, plan, s);
  // Eight waves of 16 or 32 rows, of one head each.
  hipLaunchKernelGGL((quantized_tile_kernel<DT, CT, D, D == 256 ? 1 : 2>), dim3((unsigned)(plan.workers * a.HKV)), dim3(512), 0, s, a);
  return (int)hipGetLastError();
}

// Merge workgroups up to here split their parts over 16 waves in all.
constexpr int64_t Q8_FEW_JOBS = 512;

template <int DT, int CT, int D>
int launch_quantized(QuantizedArgs a, const QuantizedPlan& plan, void* workspace, hipStream_t s) {
  const int64_t groups = plan.tiles * (plan.rows / 16);
  if (groups > 0xffffffffll / 1024) return AFA_E_SHAPE;  // a launch counts its threads in 32 bits
  const int64_t part_rows = quantized_part_rows(plan, a.HKV);
  a.workers = plan.workers;
  a.partial_o = (float*)workspace;
  a.partial_ml = a.partial_o + part_rows * D;
  a.tile_count = (uint32_t*)(a.partial_ml + part_rows * 2);
  a.records = (TileRecord*)(a.tile_count + 4);
  a.tiles = (uint32_t)plan.tiles;
  const int e = launch_form<DT, CT, D>(a, plan, s);
  if (e) return e;
  const dim3 grid((unsigned)groups, (unsigned)a.HKV);
  if (groups * a.HKV <= Q8_FEW_JOBS && D < 256)
    hipLaunchKernelGGL((quantized_merge_kernel<DT, D, D == 256 ? 1 : 256 / D>), grid, dim3(1024), 0, s, a, plan.rows / 16);
  else
    hipLaunchKernelGGL((quantized_merge_kernel<DT, D, 1>), grid, dim3(4 * D), 0, s, a, plan.rows / 16);
  return (int)hipGetLastError();
}

template <int DT, int CT>
int dispatch_quantized(const QuantizedArgs& a, int D, const QuantizedPlan& plan, void* workspace, hipStream_t s) {
  if (D == 64) return launch_quantized<DT, CT, 64>(a, plan, workspace, s);
  if (D == 128) return launch_quantized<DT, CT, 128>(a, plan, workspace, s);
  return launch_quantized<DT, CT, 256>(a, plan, workspace, s);
}

}  // namespace
}  // namespace afa

extern "C" int workspace_size_quantized_attention(uint64_t* bytes, const QuantizedParams* p) {
  using namespace afa;
  if (!bytes) return AFA_E_NULL;
  const int status = check_quantized(p);
  if (status) return status;
  *bytes = quantized_bytes(p, plan_quantized(p));
  return AFA_OK;
}

extern "C" int form_quantized_attention(int64_t form[4], const QuantizedParams* p) {
  using namespace afa;
  if (!form) return AFA_E_NULL;
  const int status = check_quantized(p);
  if (status) return status;
  const QuantizedPlan plan = plan_quantized(p);
  form[0] = plan.rows;
  form[1] = plan.heads;
  form[2] = plan.workers;
  form[3] = plan.stream ? 1 : 0;
  return AFA_OK;
}

extern "C" int launch_quantized_attention(void* stream, const void* q, const void* k_cache, const void* v_cache,
                                          const float* k_scale, const float* v_scale, const int32_t* block_table,
                                          const int32_t* cu_seqlens_q, const int32_t* seqused_kv, void* out,
                                          float* softmax_lse, void* workspace, uint64_t workspace_bytes,
                                          const QuantizedParams* p) {
  using namespace afa;
  const int status = check_quantized(p);
  if (status) return status;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !cu_seqlens_q || !seqused_kv || !out)
    return AFA_E_NULL;
  if (p->T == 0) return AFA_OK;
  if (!q8_rows_fit(q, p->q_stride_t, p->q_stride_h) || !q8_rows_fit(out, p->out_stride_t, p->out_stride_h) ||
      !q8_rows_fit(k_cache, 0, 0) || !q8_rows_fit(v_cache, 0, 0))
    return AFA_E_SHAPE;
  const QuantizedPlan plan = plan_quantized(p);
  const uint64_t need = quantized_bytes(p, plan);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return AFA_E_WORKSPACE;
  QuantizedArgs a = {};
  a.q = q;
  a.k = (const uint8_t*)k_cache;
  a.v = (const uint8_t*)v_cache;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.table = block_table;
  a.cu = cu_seqlens_q;
  a.used = seqused_kv;
  a.out = out;
  a.lse = softmax_lse;
  a.q_t = p->q_stride_t;
  a.q_h = p->q_stride_h;
  a.o_t = p->out_stride_t;
  a.o_h = p->out_stride_h;
  a.T = p->T;
  a.B = p->B;
  a.HKV = p->HKV;
  a.W = p->W;
  a.page_shift = __builtin_ctz((unsigned)p->PAGE);
  a.group_shift = __builtin_ctz((unsigned)p->GROUP);
  a.blocks = p->BLOCKS;
  a.causal = p->causal ? 1 : 0;
  a.H = p->HQ / p->HKV;
  a.scale = p->scale;
  const bool f16 = p->dtype == AFA_DTYPE_F16;
  hipStream_t s = (hipStream_t)stream;
  if (p->code == AFA_CODE_E4M3)
    return f16 ? dispatch_quantized<DT_F16, AFA_CODE_E4M3>(a, p->D, plan, workspace, s)
               : dispatch_quantized<DT_BF16, AFA_CODE_E4M3>(a, p->D, plan, workspace, s);
  return f16 ? dispatch_quantized<DT_F16, AFA_CODE_INT8>(a, p->D, plan, workspace, s)
             : dispatch_quantized<DT_BF16, AFA_CODE_INT8>(a, p->D, plan, workspace, s);
}
