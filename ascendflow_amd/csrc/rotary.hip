// Rotary positions and the append of new tokens to a paged cache, for gfx950.
//
// A pair (u, v) of columns at position p turns by the angle a = p * frequency:
//   u' = magnitude (u cos a - v sin a),  v' = magnitude (u sin a + v cos a).
// The inverse (sin -> -sin, the same magnitude) is the transposed map, so it is
// both the way back (magnitude 1) and the gradient. a reaches 10^6 radians and
// more, where a float32 angle is off by 0.03: the turns p * frequency / 2 pi are
// formed and reduced to [-1/2, 1/2] in float64 (off by 10^-7 turns at p = 2^31),
// and the cosine and sine of the rest are float32. The rotation runs in float32
// and rounds once, to the storage type.
//
// Both kernels move each byte once and are bound by HBM (few long calls) or by
// the launch and a chain of dependent loads (decode). A thread takes 8 pairs
// (two 16-byte pieces, in either layout) of a token, computes their cosines
// once and goes over several heads with them; rows that no 16-byte piece fits
// (odd widths, offsets or strides) take one pair at a time.
#include <algorithm>

#include "common.h"
#include "../../include/ascendflow_amd.h"

namespace afa {

enum { ROTARY_HALF = 0, ROTARY_INTERLEAVED = 1 };

// VEC consecutive elements of a row: 16 bytes or one element.
template <int DT, int VEC> struct Piece {
  typename B16<DT>::scalar e[VEC];
};
template <int DT, int VEC>
__device__ __forceinline__ Piece<DT, VEC> load_piece(const typename B16<DT>::scalar* p) {
  Piece<DT, VEC> out;
  if constexpr (VEC == 8) {
    const auto v = *(const typename B16<DT>::x8*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.e[i] = v[i];
  } else {
    out.e[0] = *p;
  }
  return out;
}
template <int DT, int VEC>
__device__ __forceinline__ void store_piece(typename B16<DT>::scalar* p, const Piece<DT, VEC>& v) {
  if constexpr (VEC == 8) {
    typename B16<DT>::x8 w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = v.e[i];
    *(typename B16<DT>::x8*)p = w;
  } else {
    *p = v.e[0];
  }
}

// Cosines and sines, magnitude included, of VEC pairs from `pair` on.
template <int VEC>
__device__ __forceinline__ void pair_angles(const double* frequencies, int pair, int64_t position, float magnitude,
                                            bool inverse, float (&c)[VEC], float (&s)[VEC]) {
#pragma clang fp contract(off)  // the same angles whatever VEC is
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const double turns = (double)position * (frequencies[pair + i] * 0.15915494309189535);  // 1 / 2 pi
    const float rest = (float)(turns - __builtin_rint(turns));
    float sine, cosine;
    sincospif(2.0f * rest, &sine, &cosine);
    c[i] = magnitude * cosine;
    s[i] = inverse ? -magnitude * sine : magnitude * sine;
  }
}

// Columns of the two pieces of pair group g inside the rotated part.
template <int VEC, int LAYOUT>
__device__ __forceinline__ void piece_columns(int g, int R, int& lo, int& hi) {
  if constexpr (LAYOUT == ROTARY_HALF) {
    lo = g * VEC;
    hi = lo + R / 2;
  } else {
    lo = g * 2 * VEC;
    hi = lo + VEC;
  }
}

// Rotates the VEC pairs held by the two pieces: halves pair element i of both,
// interleaved pairs neighbours (of the concatenated pieces).
template <int DT, int VEC, int LAYOUT>
__device__ __forceinline__ void rotate_pieces(Piece<DT, VEC>& lo, Piece<DT, VEC>& hi, const float (&c)[VEC],
                                              const float (&s)[VEC]) {
  typedef typename B16<DT>::scalar scalar;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    scalar* u = &lo.e[i];
    scalar* v = &hi.e[i];
    if constexpr (LAYOUT == ROTARY_INTERLEAVED && VEC > 1) {
      u = 2 * i < VEC ? &lo.e[2 * i] : &hi.e[2 * i - VEC];
      v = u + 1;
    }
    const float a = (float)*u, b = (float)*v;
    // Written as fused operations: left to the compiler, their order differs between VEC = 8 and 1.
    *u = (scalar)__builtin_fmaf(a, c[i], -(b * s[i]));
    *v = (scalar)__builtin_fmaf(a, s[i], b * c[i]);
  }
}

struct RotaryArgs {
  const void* x;
  void* out;
  const void* positions;
  const double* frequencies;
  int64_t first;  // token index of item 0 (calls of more than 2^31 items are launched in parts)
  int64_t S, x_b, x_s, x_h, out_b, out_s, out_h, position_b;
  uint32_t items;        // tokens * slots * groups of this launch
  int32_t slots, groups;  // head slots per token (head slot i takes heads i, i + slots, ...), groups per row
  int32_t rotary_groups;  // the first ones of a row; the rest copy the other columns (not in place)
  int32_t H, R, offset;
  int32_t wide_positions, inverse;
  float magnitude;
};

template <int DT, int VEC, int LAYOUT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  typedef typename B16<DT>::scalar scalar;
  const uint32_t item = blockIdx.x * 256u + threadIdx.x;
  if (item >= a.items) return;
  const uint32_t row = item / (uint32_t)a.groups;
  const int g = (int)(item - row * (uint32_t)a.groups);
  const uint32_t local = row / (uint32_t)a.slots;
  const int slot = (int)(row - local * (uint32_t)a.slots);
  const int64_t token = a.first + local;
  const int64_t b = a.S > token ? 0 : token / a.S, s = token - b * a.S;
  const scalar* x = (const scalar*)a.x + b * a.x_b + s * a.x_s;
  scalar* out = (scalar*)a.out + b * a.out_b + s * a.out_s;
  if (g >= a.rotary_groups) {
    int column = (g - a.rotary_groups) * VEC;
    if (column >= a.offset) column += a.R;
    for (int h = slot; h < a.H; h += a.slots)
      store_piece<DT, VEC>(out + h * a.out_h + column, load_piece<DT, VEC>(x + h * a.x_h + column));
    return;
  }
  const int64_t at = b * a.position_b + s;
  const int64_t position = a.wide_positions ? ((const int64_t*)a.positions)[at] : ((const int32_t*)a.positions)[at];
  float c[VEC], sn[VEC];
  pair_angles<VEC>(a.frequencies, g * VEC, position, a.magnitude, a.inverse != 0, c, sn);
  int lo, hi;
  piece_columns<VEC, LAYOUT>(g, a.R, lo, hi);
  lo += a.offset;
  hi += a.offset;
  for (int h = slot; h < a.H; h += a.slots) {
    Piece<DT, VEC> u = load_piece<DT, VEC>(x + h * a.x_h + lo), v = load_piece<DT, VEC>(x + h * a.x_h + hi);
    rotate_pieces<DT, VEC, LAYOUT>(u, v, c, sn);
    store_piece<DT, VEC>(out + h * a.out_h + lo, u);
    store_piece<DT, VEC>(out + h * a.out_h + hi, v);
  }
}

struct AppendArgs {
  const void* k;
  const void* rope;  // the rotated columns, or NULL: inside k
  const void* v;
  void* k_cache;
  void* v_cache;
  const int32_t* table;
  const int32_t* cu;
  const int32_t* used;
  const double* frequencies;
  int64_t k_t, k_h, rope_t, rope_h, v_t, v_h;
  int32_t T, B, W, PAGE, BLOCKS, HKV, DK, DV, R, offset;
  int32_t rotary_groups, copy_groups, value_groups;  // per head
  float magnitude;
};

// One wave per new token. Its request is the number of boundaries cu[1..B] at
// or below it (64 compared at a time), its position seqused - n + j; token rows
// at or past cu[B], positions outside the table's width and pages outside the
// cache write nothing.
template <int DT, int VEC, int LAYOUT>
__global__ __launch_bounds__(256) void append_paged_kv_kernel(AppendArgs a) {
  typedef typename B16<DT>::scalar scalar;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t token = (int64_t)blockIdx.x * 4 + wave;
  if (token >= a.T) return;
  int request = 0;
  for (int first = 1; first <= a.B; first += 64) {
    const int i = first + lane;
    const int below = __popcll(__ballot(i <= a.B && a.cu[min(i, a.B)] <= token));
    request += below;
    if (below < 64) break;
  }
  if (request >= a.B) return;
  const int end = a.cu[request + 1];
  const int64_t position = (int64_t)a.used[request] - end + token;
  if (position < 0) return;
  const int64_t page = position / a.PAGE;
  if (page >= a.W) return;
  const int block = a.table[(int64_t)request * a.W + page];
  if (block < 0 || block >= a.BLOCKS) return;
  const int64_t slot = (int64_t)block * a.PAGE + (position - page * a.PAGE);

  const int per_head = a.rotary_groups + a.copy_groups + a.value_groups;
  const uint32_t items = (uint32_t)per_head * (uint32_t)a.HKV;
  for (uint32_t item = lane; item < items; item += 64) {
    const int h = (int)(item / (uint32_t)per_head);
    const int g = (int)(item - (uint32_t)h * (uint32_t)per_head);
    const scalar* k = (const scalar*)a.k + token * a.k_t + h * a.k_h;
    scalar* row = (scalar*)a.k_cache + (slot * a.HKV + h) * a.DK;
    if (g < a.rotary_groups) {
      float c[VEC], s[VEC];
      pair_angles<VEC>(a.frequencies, g * VEC, position, a.magnitude, false, c, s);
      int lo, hi;
      piece_columns<VEC, LAYOUT>(g, a.R, lo, hi);
      const scalar* from = a.rope ? (const scalar*)a.rope + token * a.rope_t + h * a.rope_h : k + a.offset;
      Piece<DT, VEC> u = load_piece<DT, VEC>(from + lo), w = load_piece<DT, VEC>(from + hi);
      rotate_pieces<DT, VEC, LAYOUT>(u, w, c, s);
      store_piece<DT, VEC>(row + a.offset + lo, u);
      store_piece<DT, VEC>(row + a.offset + hi, w);
    } else if (g < a.rotary_groups + a.copy_groups) {
      int column = (g - a.rotary_groups) * VEC;
      if (column >= a.offset) column += a.R;  // with `rope` the rotated columns are the row's last: never taken
      store_piece<DT, VEC>(row + column, load_piece<DT, VEC>(k + column));
    } else {
      const int column = (g - a.rotary_groups - a.copy_groups) * VEC;
      store_piece<DT, VEC>((scalar*)a.v_cache + (slot * a.HKV + h) * a.DV + column,
                           load_piece<DT, VEC>((const scalar*)a.v + token * a.v_t + h * a.v_h + column));
    }
  }
}

namespace {

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Whether the pieces of a rotated part at `offset` fall on 16-byte groups.
bool pieces_fit(int R, int offset, int layout) {
  return offset % 8 == 0 && R % 16 == 0 && (layout == ROTARY_INTERLEAVED || (R / 2) % 8 == 0);
}

template <int DT, int VEC>
int launch_rotary(RotaryArgs a, int layout, int64_t tokens, hipStream_t s) {
  // Launches of at most 2^30 items: a token has at most H * (D / VEC) of them.
  const int64_t per_token = (int64_t)a.slots * a.groups;
  const int64_t most = std::max<int64_t>(1, (1ll << 30) / per_token);
  for (int64_t first = 0; first < tokens; first += most) {
    a.first = first;
    a.items = (uint32_t)(std::min(most, tokens - first) * per_token);
    const dim3 grid((a.items + 255u) / 256u), block(256);
    if (layout == ROTARY_HALF)
      hipLaunchKernelGGL((rotary_kernel<DT, VEC, ROTARY_HALF>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((rotary_kernel<DT, VEC, ROTARY_INTERLEAVED>), grid, block, 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return AFA_OK;
}

template <int DT, int VEC>
int launch_append(const AppendArgs& a, int layout, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + 3) / 4)), block(256);
  if (layout == ROTARY_HALF)
    hipLaunchKernelGGL((append_paged_kv_kernel<DT, VEC, ROTARY_HALF>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((append_paged_kv_kernel<DT, VEC, ROTARY_INTERLEAVED>), grid, block, 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace afa

extern "C" int launch_apply_rotary(void* stream, const void* x, const void* positions, const double* frequencies,
                                   void* out, const RotaryParams* p) {
  using namespace afa;
  if (!p || !x || !positions || !frequencies || !out) return AFA_E_NULL;
  if (p->dtype != AFA_DTYPE_BF16 && p->dtype != AFA_DTYPE_F16) return AFA_E_DTYPE;
  if (p->B < 0 || p->S < 0 || p->H <= 0 || p->D <= 0 || p->H > (1 << 20) || p->D > (1 << 16)) return AFA_E_SHAPE;
  if (p->R < 2 || p->R % 2 || p->offset < 0 || p->offset > p->D - p->R) return AFA_E_SHAPE;
  if ((p->layout != ROTARY_HALF && p->layout != ROTARY_INTERLEAVED) || (p->position_bytes != 4 && p->position_bytes != 8))
    return AFA_E_SHAPE;
  if (p->B == 0 || p->S == 0) return AFA_OK;
  if (p->B > INT64_MAX / p->S) return AFA_E_SHAPE;
  const bool in_place = x == out;
  if (in_place && (p->x_stride_b != p->out_stride_b || p->x_stride_s != p->out_stride_s || p->x_stride_h != p->out_stride_h))
    return AFA_E_SHAPE;
  const bool wide = pieces_fit(p->R, p->offset, p->layout) && (in_place || p->D % 8 == 0) && on16(x) && on16(out) &&
                    (p->x_stride_b | p->x_stride_s | p->x_stride_h | p->out_stride_b | p->out_stride_s | p->out_stride_h) % 8 == 0;
  const int vec = wide ? 8 : 1;
  RotaryArgs a;
  a.x = x;
  a.out = out;
  a.positions = positions;
  a.frequencies = frequencies;
  a.S = p->S;
  a.x_b = p->x_stride_b;
  a.x_s = p->x_stride_s;
  a.x_h = p->x_stride_h;
  a.out_b = p->out_stride_b;
  a.out_s = p->out_stride_s;
  a.out_h = p->out_stride_h;
  a.position_b = p->position_stride_b;
  a.rotary_groups = p->R / 2 / vec;
  a.groups = a.rotary_groups + (in_place ? 0 : (p->D - p->R) / vec);
  a.H = p->H;
  a.R = p->R;
  a.offset = p->offset;
  a.wide_positions = p->position_bytes == 8;
  a.inverse = p->inverse ? 1 : 0;
  a.magnitude = p->magnitude;
  // Heads per thread: as many share a thread's cosines as leave two waves per SIMD.
  const int64_t tokens = p->B * p->S;
  int heads = 1;
  while (heads < 8 && heads < p->H && tokens * ((p->H + 2 * heads - 1) / (2 * heads)) * a.groups >= 256ll * 512) heads *= 2;
  a.slots = (p->H + heads - 1) / heads;
  if ((int64_t)a.slots * a.groups > (1ll << 30)) return AFA_E_SHAPE;
  hipStream_t s = (hipStream_t)stream;
  if (p->dtype == AFA_DTYPE_F16)
    return wide ? launch_rotary<DT_F16, 8>(a, p->layout, tokens, s) : launch_rotary<DT_F16, 1>(a, p->layout, tokens, s);
  return wide ? launch_rotary<DT_BF16, 8>(a, p->layout, tokens, s) : launch_rotary<DT_BF16, 1>(a, p->layout, tokens, s);
}

extern "C" int launch_append_paged_kv(void* stream, const void* k, const void* rope, const void* v,
                                      const int32_t* block_table, const int32_t* cu_seqlens_q, const int32_t* seqused_kv,
                                      const double* frequencies, void* k_cache, void* v_cache,
                                      const AppendPagedKvParams* p) {
  using namespace afa;
  if (!p) return AFA_E_NULL;
  if (p->dtype != AFA_DTYPE_BF16 && p->dtype != AFA_DTYPE_F16) return AFA_E_DTYPE;
  if (p->T < 0 || p->B <= 0 || p->W <= 0 || p->PAGE <= 0 || p->BLOCKS <= 0 || p->HKV <= 0 || p->DK <= 0 || p->DV < 0)
    return AFA_E_SHAPE;
  if (p->HKV > (1 << 16) || p->DK > (1 << 14) || p->DV > (1 << 14)) return AFA_E_SHAPE;
  if (p->R < 0 || p->R % 2 || p->offset < 0 || p->R > p->DK || p->offset > p->DK - p->R) return AFA_E_SHAPE;
  if (p->layout != ROTARY_HALF && p->layout != ROTARY_INTERLEAVED) return AFA_E_SHAPE;
  if (rope && (p->R == 0 || p->offset != p->DK - p->R)) return AFA_E_SHAPE;
  if (!block_table || !cu_seqlens_q || !seqused_kv || !k_cache || (p->R > 0 && !frequencies)) return AFA_E_NULL;
  if ((!k && !(rope && p->R == p->DK)) || (p->DV > 0 && (!v || !v_cache))) return AFA_E_NULL;
  if (p->T == 0) return AFA_OK;
  const int R = p->R;
  bool wide = p->DK % 8 == 0 && p->DV % 8 == 0 && (R == 0 || pieces_fit(R, p->offset, p->layout)) && on16(k) &&
              on16(k_cache) && (p->k_stride_t | p->k_stride_h) % 8 == 0;
  if (rope) wide = wide && on16(rope) && (p->rope_stride_t | p->rope_stride_h) % 8 == 0;
  if (p->DV) wide = wide && on16(v) && on16(v_cache) && (p->v_stride_t | p->v_stride_h) % 8 == 0;
  const int vec = wide ? 8 : 1;
  AppendArgs a;
  a.k = k;
  a.rope = rope;
  a.v = v;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.table = block_table;
  a.cu = cu_seqlens_q;
  a.used = seqused_kv;
  a.frequencies = frequencies;
  a.k_t = p->k_stride_t;
  a.k_h = p->k_stride_h;
  a.rope_t = p->rope_stride_t;
  a.rope_h = p->rope_stride_h;
  a.v_t = p->v_stride_t;
  a.v_h = p->v_stride_h;
  a.T = p->T;
  a.B = p->B;
  a.W = p->W;
  a.PAGE = p->PAGE;
  a.BLOCKS = p->BLOCKS;
  a.HKV = p->HKV;
  a.DK = p->DK;
  a.DV = p->DV;
  a.R = R;
  a.offset = p->offset;
  a.rotary_groups = R / 2 / vec;
  a.copy_groups = (p->DK - R) / vec;
  a.value_groups = p->DV / vec;
  a.magnitude = p->magnitude;
  hipStream_t s = (hipStream_t)stream;
  if (p->dtype == AFA_DTYPE_F16)
    return wide ? launch_append<DT_F16, 8>(a, p->layout, s) : launch_append<DT_F16, 1>(a, p->layout, s);
  return wide ? launch_append<DT_BF16, 8>(a, p->layout, s) : launch_append<DT_BF16, 1>(a, p->layout, s);
}
