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
// (append writes none below), which keeps every ratio of them inside float32.
//
// The sums, the maximum and the output are float32; p is rounded to the query's type (a
// matrix operand has to be), at most half a step of each weight, while the denominator
// sums the weights before rounding. float16 raises the maximum only when it grows by more
// than 2^8, bfloat16, whose step is coarser, whenever it grows.
#include <algorithm>
#include <cmath>

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
  int32_t workers;          // workgroups of a key/value head
  float* partial_o;         // [2 * workers][HKV][ROWS][D], not normalised
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

// ---- stream form ---------------------------------------------------------------
//
// For the few rows of decode and verification: a tile is 16 QT packed rows of one
// key/value head, a chunk 128 cache rows, 32 for each of four waves. Waves are on their
// own until a tile ends: no barrier, no LDS; each keeps all rows' queries and an output of
// its own, and its codes go from memory to registers, a chunk ahead of their use.
// S^T[keys, rows] = K Q^T: a lane loads 16 bytes of a key row (the order of columns is
// free, queries follow it). O^T[columns, rows] += V^T P^T: lane (g, i) needs a column's
// values of the eight keys that its P holds, which lie a row apart, so it loads D / 16
// columns of those eight rows and transposes bytes in registers; the tiles of columns
// that come out interleave, which leaves each lane with D / 4 consecutive ones.
template <int QT> struct StreamForm {
  static constexpr int ROWS = 16 * QT, KEYS = 128, THREADS = 256;
  static constexpr uint32_t START = 1, LEAST = 2;
  static constexpr float JOIN = 4.0f;
};

template <int BYTES> struct Bytes;
template <> struct Bytes<4> { typedef uint32_t type __attribute__((ext_vector_type(1))); };
template <> struct Bytes<8> { typedef u32x2 type; };
template <> struct Bytes<16> { typedef u32x4 type; };

// 4 x 4 bytes, rows to columns.
__device__ __forceinline__ void transpose4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t* c) {
  const uint32_t a = __builtin_amdgcn_perm(r1, r0, 0x05010400u), b = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
  const uint32_t d = __builtin_amdgcn_perm(r3, r2, 0x05010400u), e = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
  c[0] = __builtin_amdgcn_perm(d, a, 0x05040100u);
  c[1] = __builtin_amdgcn_perm(d, a, 0x07060302u);
  c[2] = __builtin_amdgcn_perm(e, b, 0x05040100u);
  c[3] = __builtin_amdgcn_perm(e, b, 0x07060302u);
}

template <int DT, int CT, int D, int QT>
__global__ __launch_bounds__(256, 2) void quantized_stream_kernel(QuantizedArgs a) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x8 x8;
  typedef StreamForm<QT> F;
  typedef typename Bytes<D / 16>::type vbytes;
  constexpr int ROWS = F::ROWS, KEYS = F::KEYS, KL = D / 64, VT = D / 16;
  __shared__ f32x4 joined_o[4][VT][64];
  __shared__ float2 joined_ml[4][16];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, i16 = lane & 15;
  const int H = a.H;
  const int kv_head = uniform((int)(blockIdx.x % (uint32_t)a.HKV));
  const uint32_t worker = (uint32_t)uniform((int)(blockIdx.x / (uint32_t)a.HKV));

  TileShare share;
  if (!find_share<F>(a, worker, worker, share)) return;
  int request = share.request;
  uint32_t place = share.place, offset = share.offset;
  uint64_t left = share.end - share.begin;
  const float scale_log2 = a.scale * LOG2E;
  const uint32_t row_bytes = (uint32_t)a.HKV * D;
  const uint32_t k_off = (uint32_t)i16 * row_bytes + 16u * g, v_off = (uint32_t)(4 * g) * row_bytes + (uint32_t)(VT * i16);

  for (;;) {
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
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m_run[qt] = -1e30f;  // finite: a chunk that hides all its keys gives p = 0, never NaN
      l_run[qt] = 0.f;
#pragma unroll
      for (int c = 0; c < VT; ++c) o[qt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    struct Part {  // a wave's 32 rows of a chunk
      u32x4 k[2][KL];
      vbytes v[8];
      float ks[2], vs[2];
      uint32_t good;  // bit t: the page of 16-row group t holds keys
    };
    const const_ints pages = constant(a.table + (int64_t)request * a.W);
    const int page_mask = (1 << a.page_shift) - 1;
    int page[2];  // of the next part to load, -1 past the end
    auto look_up = [&](int chunk) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = chunk * KEYS + wave * 32 + 16 * t;
        page[t] = chunk < chunks && key < kv_end ? pages[key >> a.page_shift] : -1;
      }
    };
    typedef const __attribute__((address_space(4))) float* const_floats;
    auto load = [&](int chunk, Part& p) {
      p.good = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = chunk * KEYS + wave * 32 + 16 * t;
        const bool inside = (uint32_t)page[t] < (uint32_t)a.blocks;
        p.good |= inside ? 1u << t : 0u;
        // Rows that are not there read the cache's first ones instead (hidden later).
        const int64_t row = inside ? ((int64_t)page[t] << a.page_shift) + (key & page_mask) : 0;
        const int64_t at = row * row_bytes + kv_head * D;
        const uint8_t* k = a.k + at;
        const uint8_t* v = a.v + at;
        const int64_t block = (row >> a.group_shift) * a.HKV + kv_head;
        p.ks[t] = ((const_floats)(uintptr_t)a.k_scale)[block];
        p.vs[t] = ((const_floats)(uintptr_t)a.v_scale)[block];
#pragma unroll
        for (int l = 0; l < KL; ++l) p.k[t][l] = *(const u32x4*)(k + (k_off + 64u * l));
#pragma unroll
        for (int r = 0; r < 4; ++r) p.v[4 * t + r] = *(const vbytes*)(v + (v_off + (uint32_t)r * row_bytes));
      }
    };
    auto attend = [&](int chunk, Part& p) {
      const int key0 = chunk * KEYS + wave * 32;
      if (key0 >= kv_end) return;
      f32x4 s[2][QT];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[t][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int l = 0; l < KL; ++l)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const x8 kf = Codes<DT, CT>::decode(p.k[t][l][2 * h], p.k[t][l][2 * h + 1]);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) s[t][qt] = B16<DT>::mfma(kf, qf[qt][2 * l + h], s[t][qt]);
          }
      }
      if (key0 + 32 > clean_end || p.good != 3u) {  // uniform
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = 16 * t + 4 * g + r;
            const bool page_holds = (p.good >> t) & 1u;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) s[t][qt][r] = page_holds && key0 + key < limit[qt] ? s[t][qt][r] : -INFINITY;
            // Values that nobody sees may be codes of no number, which no weight of 0 would hide.
            if (!(page_holds && key0 + key < kv_end)) p.v[4 * t + r] = vbytes(0);
          }
      }
      float sk[2], lv[2], iv[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool page_holds = (p.good >> t) & 1u;  // else the scales are those of other rows
        const float ks = page_holds ? p.ks[t] : 1.0f, vs = page_holds ? at_least(p.vs[t], Q8_LEAST_SCALE) : 1.0f;
        sk[t] = at_least(ks * scale_log2, 1.17549435e-38f);  // not 0: times a hidden score
        lv[t] = __log2f(vs);
        iv[t] = 1.0f / vs;
      }
      x8 pf[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float mine = fmaxf(fmaxf(s[t][qt][0], s[t][qt][1]), fmaxf(s[t][qt][2], s[t][qt][3]));
          top = fmaxf(top, __builtin_fmaf(mine, sk[t], lv[t]));
        }
        const float m_new = fmaxf(m_run[qt], max_over_lane_groups(top));
        if (__ballot(m_new > m_run[qt] + q8_tau<DT>()) != 0ull) {
          const float alpha = fast_exp2(m_run[qt] - m_new);
          l_run[qt] *= alpha;
#pragma unroll
          for (int c = 0; c < VT; ++c) o[qt][c] *= alpha;
          m_run[qt] = m_new;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float shift = lv[t] - m_run[qt];
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = fast_exp2(__builtin_fmaf(s[t][qt][r], sk[t], shift));
            sum += w;
            pf[qt][4 * t + r] = (scalar)w;
          }
          l_run[qt] = __builtin_fmaf(sum, iv[t], l_run[qt]);
        }
      }
#pragma unroll
      for (int w = 0; w < VT / 4; ++w) {
        uint32_t lo[4], hi[4];
        transpose4(p.v[0][w], p.v[1][w], p.v[2][w], p.v[3][w], lo);
        transpose4(p.v[4][w], p.v[5][w], p.v[6][w], p.v[7][w], hi);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const x8 vf = Codes<DT, CT>::decode(lo[c], hi[c]);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) o[qt][4 * w + c] = B16<DT>::mfma(vf, pf[qt], o[qt][4 * w + c]);
        }
      }
    };

    Part even, odd;
    look_up(begin);
    if (begin < chunks) load(begin, even);
    look_up(begin + 1);
    for (int c = begin; c < chunks; c += 2) {
      if (c + 1 < chunks) load(c + 1, odd);
      look_up(c + 2);
      attend(c, even);
      if (c + 1 < chunks) {
        if (c + 2 < chunks) load(c + 2, even);
        look_up(c + 3);
        attend(c + 1, odd);
      }
    }

    // The four waves' sums, 16 rows at a time. Lane (g, i) of column tile c, element r holds
    // column VT (4 g + r) + c of row i; here a thread takes VT columns of a row.
    const int row_of = tid & 15, unit = tid >> 4;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      __syncthreads();  // the last round's are read
      const float total = sum_over_lane_groups(l_run[qt]);
#pragma unroll
      for (int c = 0; c < VT; ++c) joined_o[wave][c][lane] = o[qt][c];
      if (g == 0) joined_ml[wave][i16] = make_float2(m_run[qt], total);
      __syncthreads();
      const int row = (int)tile * ROWS + qt * 16 + row_of;
      if (row < rows) {
        float2 ml[4];
        float top = -1e30f, sum = 0.f, weight[4], acc[VT];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          ml[w] = joined_ml[w][row_of];
          top = fmaxf(top, ml[w].x);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          weight[w] = fast_exp2(ml[w].x - top);
          sum = __builtin_fmaf(weight[w], ml[w].y, sum);
        }
#pragma unroll
        for (int c = 0; c < VT; ++c) {
          acc[c] = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            acc[c] = __builtin_fmaf(weight[w], ((const float*)&joined_o[w][c][(unit >> 2) * 16 + row_of])[unit & 3], acc[c]);
        }
        if (whole) {
          const float inv = sum > 0.f ? 1.0f / sum : 0.f;
          const int token = row / H, head = kv_head * H + row - token * H;
          scalar v[VT];
#pragma unroll
          for (int c = 0; c < VT; ++c) v[c] = (scalar)(acc[c] * inv);
          scalar* out = (scalar*)a.out + (int64_t)(start + token) * a.o_t + (int64_t)head * a.o_h + VT * unit;
          __builtin_memcpy(__builtin_assume_aligned(out, 2 * VT < 16 ? 2 * VT : 16), v, sizeof(v));
          if (a.lse && unit == 0) a.lse[(int64_t)(start + token) * (a.HKV * H) + head] = row_lse(top, sum);
        } else {
          const int64_t at = ((2 * (int64_t)worker + (offset == 0 ? 1 : 0)) * a.HKV + kv_head) * ROWS + qt * 16 + row_of;
          __builtin_memcpy(__builtin_assume_aligned(a.partial_o + at * D + VT * unit, 16), acc, sizeof(acc));
          if (unit == 0) *(float2*)(a.partial_ml + at * 2) = make_float2(top, sum);
        }
      }
    }
    if (left == 0) return;
    offset = 0;
    ++place;
  }
}

// Combines the parts of the tiles that several workgroups share, in order:
// out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p. 16 rows of a head a workgroup.
template <int DT, int D>
__global__ __launch_bounds__(256) void quantized_merge_kernel(QuantizedArgs a, int tile_rows) {
  typedef typename B16<DT>::scalar scalar;
  constexpr int VT = D / 16, AHEAD = 4;
  const uint32_t groups = (uint32_t)tile_rows / 16;
  const uint32_t tile = blockIdx.x / groups, group = blockIdx.x % groups;
  const int kv_head = blockIdx.y;
  if (tile >= *constant((const int32_t*)a.tile_count)) return;
  const TileRecord record = a.records[tile];
  const int row_of = (int)group * 16 + (threadIdx.x & 15), unit = threadIdx.x >> 4;
  if (record.first == record.last || row_of >= record.rows) return;
  const int parts = record.last - record.first + 1;
  auto slot = [&](int p) {
    return ((2 * (int64_t)(record.first + p) + (p == 0 ? 1 : 0)) * a.HKV + kv_head) * tile_rows + row_of;
  };
  float top = -1e30f, total = 0.f, acc[VT];
  for (int p = 0; p < parts; ++p) top = fmaxf(top, a.partial_ml[slot(p) * 2]);
#pragma unroll
  for (int c = 0; c < VT; ++c) acc[c] = 0.f;
  for (int p = 0; p < parts; p += AHEAD) {
    float2 ml[AHEAD];
    f32x4 v[AHEAD][VT / 4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int64_t at = slot(min(p + i, parts - 1));
      ml[i] = *(const float2*)(a.partial_ml + at * 2);
#pragma unroll
      for (int j = 0; j < VT / 4; ++j) v[i][j] = *(const f32x4*)(a.partial_o + at * D + VT * unit + 4 * j);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float weight = p + i < parts ? fast_exp2(ml[i].x - top) : 0.f;
      total = __builtin_fmaf(weight, ml[i].y, total);
#pragma unroll
      for (int c = 0; c < VT; ++c) acc[c] = __builtin_fmaf(weight, v[i][c / 4][c % 4], acc[c]);
    }
  }
  const int packed = record.row + row_of, token = packed / a.H, head = kv_head * a.H + packed - token * a.H;
  const float inv = total > 0.f ? 1.0f / total : 0.f;
  scalar v[VT];
#pragma unroll
  for (int c = 0; c < VT; ++c) v[c] = (scalar)(acc[c] * inv);
  scalar* out = (scalar*)a.out + (int64_t)(record.start + token) * a.o_t + (int64_t)head * a.o_h + VT * unit;
  __builtin_memcpy(__builtin_assume_aligned(out, 2 * VT < 16 ? 2 * VT : 16), v, sizeof(v));
  if (a.lse && unit == 0) a.lse[(int64_t)(record.start + token) * (a.HKV * a.H) + head] = row_lse(top, total);
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
  // Packed rows, tiles, positions and the offsets of 64 cache rows are 32-bit numbers.
  if ((int64_t)p->T * p->HQ > 0x7fffff00ll || (int64_t)p->W * p->PAGE > 0x7fffff00ll || p->B > 0x3fffffff) return AFA_E_SHAPE;
  if (p->HKV > 32768) return AFA_E_SHAPE;
  if (!(p->scale > 0.0f) || !std::isfinite(p->scale)) return AFA_E_SHAPE;
  return AFA_OK;
}

constexpr int Q8_SLOTS = 512;  // workgroups of four waves that the GPU holds

struct QuantizedPlan {
  int rows;       // of a tile
  int workers;    // per key/value head
  int64_t tiles;  // the most that monotone cu_seqlens_q can give
};
QuantizedPlan plan_quantized(const QuantizedParams* p) {
  const int64_t H = p->HQ / p->HKV;
  QuantizedPlan plan;
  plan.rows = ((int64_t)p->T + p->B - 1) / p->B * H > 16 ? 32 : 16;
  plan.workers = std::max(1, Q8_SLOTS / p->HKV);
  plan.tiles = p->T * H / plan.rows + p->B;
  return plan;
}
int64_t quantized_part_rows(const QuantizedPlan& plan, int HKV) { return 2ll * plan.workers * HKV * plan.rows; }
uint64_t quantized_bytes(const QuantizedParams* p, const QuantizedPlan& plan) {
  if (p->T == 0) return 0;
  return (uint64_t)(quantized_part_rows(plan, p->HKV) * (p->D + 2) * 4 + plan.tiles * (int64_t)sizeof(TileRecord) + 16);
}

template <int DT, int CT, int D>
int launch_quantized(QuantizedArgs a, const QuantizedPlan& plan, void* workspace, hipStream_t s) {
  const int64_t groups = plan.tiles * (plan.rows / 16);
  if (groups > 0xffffffffll / 256) return AFA_E_SHAPE;  // a launch counts its threads in 32 bits
  const int64_t part_rows = quantized_part_rows(plan, a.HKV);
  a.workers = plan.workers;
  a.partial_o = (float*)workspace;
  a.partial_ml = a.partial_o + part_rows * D;
  a.tile_count = (uint32_t*)(a.partial_ml + part_rows * 2);
  a.records = (TileRecord*)(a.tile_count + 4);
  a.tiles = (uint32_t)plan.tiles;
  const dim3 grid((unsigned)(plan.workers * a.HKV));
  if (plan.rows == 16)
    hipLaunchKernelGGL((quantized_stream_kernel<DT, CT, D, 1>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((quantized_stream_kernel<DT, CT, D, 2>), grid, dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL((quantized_merge_kernel<DT, D>), dim3((unsigned)groups, (unsigned)a.HKV), dim3(256), 0, s, a, plan.rows);
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

extern "C" int form_quantized_attention(int64_t form[2], const QuantizedParams* p) {
  using namespace afa;
  if (!form) return AFA_E_NULL;
  const int status = check_quantized(p);
  if (status) return status;
  const QuantizedPlan plan = plan_quantized(p);
  form[0] = plan.rows;
  form[1] = plan.workers;
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
