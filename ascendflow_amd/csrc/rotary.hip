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
// Both kernels move each byte once and are bound by HBM (many tokens) or by the
// launch and a chain of dependent loads (decode). A workgroup takes a few
// tokens: it works out their cosines and sines once, one pair a thread, into
// LDS, then goes over the rows in pieces of 8 pairs (two 16-byte accesses, in
// either layout); rows that no 16-byte piece fits (odd widths, offsets or
// strides) are taken one pair at a time. 8192 tokens of 64 heads x 64 columns take
// 27.6 us (4.9 TB/s, the rate of a large copy), 4209 ragged prompt tokens of 8
// heads x 256 columns into pages 11.9 us (22.5 where each thread worked out the
// cosines of its own 8 pairs), 384 decode tokens of one 576-column row 3.9 (6.1).
#include <algorithm>
#include <cmath>

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

constexpr int ROT_MAX_PAIRS = 512, ROT_TOKENS = 8;  // pairs of a row, tokens of a workgroup
constexpr int ROT_LDS_PAIRS = 1024;                 // pairs of all its tokens
constexpr int ROT_MAX_D = 16384;                    // columns of a row
constexpr int ROT_MAX_HKV = 32768;                  // heads of a cache
// Workgroups of 256 threads along one dimension of a grid, whose threads a launch
// counts in 32 bits: a call with more of them has further slices.
constexpr int64_t ROT_SLICE = 1 << 23;

// Cosine and sine of a pair, magnitude included.
__device__ __forceinline__ float2 pair_angle(double frequency, int64_t position, float magnitude, bool inverse) {
#pragma clang fp contract(off)
  const double turns = (double)position * (frequency * 0.15915494309189535);  // 1 / 2 pi
  const float rest = (float)(turns - __builtin_rint(turns));
  float sine, cosine;
  sincospif(2.0f * rest, &sine, &cosine);
  return make_float2(magnitude * cosine, inverse ? -magnitude * sine : magnitude * sine);
}

// index / n for index * n < 2^32, with m = ceil(2^32 / n): the product exceeds
// index / n by index (m n - 2^32) / (2^32 n) < 1 / n. n = 1 has m = 0.
__device__ __forceinline__ uint32_t divide(uint32_t index, uint32_t m) { return m ? __umulhi(index, m) : index; }

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
__device__ __forceinline__ void rotate_pieces(Piece<DT, VEC>& lo, Piece<DT, VEC>& hi, const float2* angles) {
  typedef typename B16<DT>::scalar scalar;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    scalar* u = &lo.e[i];
    scalar* v = &hi.e[i];
    if constexpr (LAYOUT == ROTARY_INTERLEAVED && VEC > 1) {
      u = 2 * i < VEC ? &lo.e[2 * i] : &hi.e[2 * i - VEC];
      v = u + 1;
    }
    const float2 t = angles[i];
    const float a = (float)*u, b = (float)*v;
    // Written as fused operations: left to the compiler, their order differs between VEC = 8 and 1.
    *u = (scalar)__builtin_fmaf(a, t.x, -(b * t.y));
    *v = (scalar)__builtin_fmaf(a, t.y, b * t.x);
  }
}

struct RotaryArgs {
  const void* x;
  void* out;
  const void* positions;
  const double* frequencies;
  int64_t tokens, S, x_b, x_s, x_h, out_b, out_s, out_h, position_b;
  int32_t block_tokens, block_heads, head_blocks;  // of a workgroup; workgroups per token block
  int32_t groups;         // pieces of a row: the rotated ones, then (not in place) the other columns
  int32_t rotary_groups;
  uint32_t groups_m, heads_m;  // for divide(): by groups, by block_heads
  int32_t H, R, offset;
  int32_t wide_positions, inverse;
  float magnitude;
};

template <int DT, int VEC, int LAYOUT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  typedef typename B16<DT>::scalar scalar;
  __shared__ float2 angles[ROT_LDS_PAIRS];
  const int pairs = a.R / 2;
  const uint32_t block = blockIdx.y * (uint32_t)ROT_SLICE + blockIdx.x;
  const int64_t token0 = (int64_t)(block / (uint32_t)a.head_blocks) * a.block_tokens;
  const int head0 = (int)(block % (uint32_t)a.head_blocks) * a.block_heads;
  if (token0 >= a.tokens) return;  // the last slice's end
  const int tokens = (int)min((int64_t)a.block_tokens, a.tokens - token0);
  auto place = [&](int t, int64_t& b, int64_t& s) {
    const int64_t token = token0 + t;
    b = a.S > token ? 0 : token / a.S;
    s = token - b * a.S;
  };
  for (int i = threadIdx.x; i < tokens * pairs; i += 256) {
    const int t = i / pairs;
    int64_t b, s;
    place(t, b, s);
    const int64_t at = b * a.position_b + s;
    const int64_t position = a.wide_positions ? ((const int64_t*)a.positions)[at] : ((const int32_t*)a.positions)[at];
    angles[i] = pair_angle(a.frequencies[i - t * pairs], position, a.magnitude, a.inverse != 0);
  }
  __syncthreads();
  const uint32_t items = (uint32_t)(tokens * a.block_heads * a.groups);
  for (uint32_t item = threadIdx.x; item < items; item += 256) {
    const uint32_t row = divide(item, a.groups_m), t = divide(row, a.heads_m);
    const int g = (int)(item - row * (uint32_t)a.groups), h = head0 + (int)(row - t * (uint32_t)a.block_heads);
    if (h >= a.H) continue;
    int64_t b, s;
    place((int)t, b, s);
    const scalar* x = (const scalar*)a.x + b * a.x_b + s * a.x_s + h * a.x_h;
    scalar* out = (scalar*)a.out + b * a.out_b + s * a.out_s + h * a.out_h;
    if (g < a.rotary_groups) {
      int lo, hi;
      piece_columns<VEC, LAYOUT>(g, a.R, lo, hi);
      lo += a.offset;
      hi += a.offset;
      Piece<DT, VEC> u = load_piece<DT, VEC>(x + lo), v = load_piece<DT, VEC>(x + hi);
      rotate_pieces<DT, VEC, LAYOUT>(u, v, angles + (int)t * pairs + g * VEC);
      store_piece<DT, VEC>(out + lo, u);
      store_piece<DT, VEC>(out + hi, v);
    } else {
      int column = (g - a.rotary_groups) * VEC;
      if (column >= a.offset) column += a.R;
      store_piece<DT, VEC>(out + column, load_piece<DT, VEC>(x + column));
    }
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
  int32_t block_tokens, block_heads;  // of a workgroup
  int32_t rotary_groups, copy_groups, groups;  // pieces per head: rotated, other key columns, all (the values' last)
  uint32_t groups_m, heads_m;                  // for divide(): by groups, by block_heads
  float magnitude;
};

// A workgroup of four waves takes block_tokens new tokens, with all heads but
// for rows so wide that divide() cannot hold them all. One wave finds a
// token's place: its request is the number of boundaries cu[1..B] at or below
// it (64 compared at a time), its position seqused - n + j; token rows below cu[0], at
// or past cu[B], positions outside the table's width and pages outside the cache have none.
template <int DT, int VEC, int LAYOUT>
__global__ __launch_bounds__(256) void append_paged_kv_kernel(AppendArgs a) {
  typedef typename B16<DT>::scalar scalar;
  __shared__ float2 angles[ROT_LDS_PAIRS];
  __shared__ int64_t slots[ROT_TOKENS], positions[ROT_TOKENS];  // cache row, -1: none
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t token0 = (blockIdx.z * ROT_SLICE + blockIdx.x) * a.block_tokens;
  if (token0 >= a.T) return;  // the last slice's end
  const int tokens = (int)min((int64_t)a.block_tokens, (int64_t)a.T - token0);
  const int pairs = a.R / 2;
  auto find = [&](int64_t token, int64_t& position) -> int64_t {
    int request = 0;
    for (int first = 1; first <= a.B; first += 64) {
      const int i = first + lane;
      const int below = __popcll(__ballot(i <= a.B && a.cu[min(i, a.B)] <= token));
      request += below;
      if (below < 64) break;
    }
    position = -1;
    if (request >= a.B || token < a.cu[0]) return -1;
    position = (int64_t)a.used[request] - a.cu[request + 1] + token;
    if (position < 0) return -1;
    const int64_t page = position / a.PAGE;
    if (page >= a.W) return -1;
    const int block = a.table[(int64_t)request * a.W + page];
    if (block < 0 || block >= a.BLOCKS) return -1;
    return (int64_t)block * a.PAGE + (position - page * a.PAGE);
  };
  for (int t = wave; t < tokens; t += 4) {
    int64_t position;
    const int64_t slot = find(token0 + t, position);
    if (lane == 0) {
      slots[t] = slot;
      positions[t] = position;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * pairs; i += 256) {
    const int t = i / pairs;
    angles[i] = pair_angle(a.frequencies[i - t * pairs], positions[t], a.magnitude, false);
  }
  __syncthreads();
  const int head0 = (int)blockIdx.y * a.block_heads;
  const uint32_t items = (uint32_t)(tokens * a.block_heads * a.groups);
  for (uint32_t item = threadIdx.x; item < items; item += 256) {
    const uint32_t head_row = divide(item, a.groups_m), t = divide(head_row, a.heads_m);
    const int g = (int)(item - head_row * (uint32_t)a.groups), h = head0 + (int)(head_row - t * (uint32_t)a.block_heads);
    const int64_t slot = slots[t], token = token0 + t;
    if (slot < 0 || h >= a.HKV) continue;
    const scalar* k = (const scalar*)a.k + token * a.k_t + h * a.k_h;
    scalar* row = (scalar*)a.k_cache + (slot * a.HKV + h) * a.DK;
    if (g < a.rotary_groups) {
      int lo, hi;
      piece_columns<VEC, LAYOUT>(g, a.R, lo, hi);
      const scalar* from = a.rope ? (const scalar*)a.rope + token * a.rope_t + h * a.rope_h : k + a.offset;
      Piece<DT, VEC> u = load_piece<DT, VEC>(from + lo), w = load_piece<DT, VEC>(from + hi);
      rotate_pieces<DT, VEC, LAYOUT>(u, w, angles + (int)t * pairs + g * VEC);
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

// Multiplier of divide() for n.
uint32_t divider(int64_t n) { return n == 1 ? 0u : (uint32_t)(((1ull << 32) + n - 1) / n); }

template <int DT, int VEC>
int launch_rotary(const RotaryArgs& a, int layout, int64_t blocks, hipStream_t s) {
  const dim3 grid((unsigned)std::min(blocks, ROT_SLICE), (unsigned)((blocks + ROT_SLICE - 1) / ROT_SLICE)), block(256);
  if (layout == ROTARY_HALF)
    hipLaunchKernelGGL((rotary_kernel<DT, VEC, ROTARY_HALF>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((rotary_kernel<DT, VEC, ROTARY_INTERLEAVED>), grid, block, 0, s, a);
  return (int)hipGetLastError();
}

template <int DT, int VEC>
int launch_append(const AppendArgs& a, int layout, hipStream_t s) {
  const int64_t blocks = ((int64_t)a.T + a.block_tokens - 1) / a.block_tokens;
  const dim3 grid((unsigned)std::min(blocks, ROT_SLICE), (unsigned)((a.HKV + a.block_heads - 1) / a.block_heads),
                  (unsigned)((blocks + ROT_SLICE - 1) / ROT_SLICE));
  const dim3 block(256);
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
  if (p->B < 0 || p->S < 0 || p->H <= 0 || p->D <= 0 || p->D > ROT_MAX_D || p->R > 2 * ROT_MAX_PAIRS) return AFA_E_SHAPE;
  if (p->R < 2 || p->R % 2 || p->offset < 0 || p->offset > p->D - p->R) return AFA_E_SHAPE;
  if ((p->layout != ROTARY_HALF && p->layout != ROTARY_INTERLEAVED) || (p->position_bytes != 4 && p->position_bytes != 8))
    return AFA_E_SHAPE;
  if (!std::isfinite(p->magnitude)) return AFA_E_SHAPE;
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
  // Workgroups of a few tokens and all heads (at most 2^15 pieces, which
  // divide() holds), of fewer heads, then of fewer tokens, until there are four
  // per CU.
  const int64_t tokens = p->B * p->S;
  int64_t block_tokens = std::min<int64_t>(ROT_TOKENS, ROT_LDS_PAIRS / (p->R / 2));
  int64_t heads = std::min<int64_t>(p->H, std::max<int64_t>(1, (1 << 15) / (block_tokens * a.groups)));
  auto count = [&] { return (tokens + block_tokens - 1) / block_tokens * ((p->H + heads - 1) / heads); };
  while (heads > 1 && count() < 1024) heads = (heads + 1) / 2;
  while (block_tokens > 1 && (count() < 1024 || block_tokens * heads * a.groups > (1 << 15))) block_tokens /= 2;
  if (count() > 0x7fffffffll) return AFA_E_SHAPE;
  a.tokens = tokens;
  a.block_tokens = (int32_t)block_tokens;
  a.block_heads = (int32_t)heads;
  a.head_blocks = (int32_t)((p->H + heads - 1) / heads);
  a.groups_m = divider(a.groups);
  a.heads_m = divider(heads);
  hipStream_t s = (hipStream_t)stream;
  if (p->dtype == AFA_DTYPE_F16)
    return wide ? launch_rotary<DT_F16, 8>(a, p->layout, count(), s) : launch_rotary<DT_F16, 1>(a, p->layout, count(), s);
  return wide ? launch_rotary<DT_BF16, 8>(a, p->layout, count(), s) : launch_rotary<DT_BF16, 1>(a, p->layout, count(), s);
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
  if (p->HKV > ROT_MAX_HKV) return AFA_E_SHAPE;
  if (p->DK > ROT_MAX_D || p->DV > ROT_MAX_D || p->R > 2 * ROT_MAX_PAIRS) return AFA_E_SHAPE;
  if (p->R < 0 || p->R % 2 || p->offset < 0 || p->R > p->DK || p->offset > p->DK - p->R) return AFA_E_SHAPE;
  if (p->layout != ROTARY_HALF && p->layout != ROTARY_INTERLEAVED) return AFA_E_SHAPE;
  if (!std::isfinite(p->magnitude)) return AFA_E_SHAPE;
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
  a.groups = a.rotary_groups + a.copy_groups + p->DV / vec;
  // One token a workgroup up to four workgroups per CU, then up to eight; fewer,
  // then fewer heads (at most 2^15 groups leave three), until divide() holds
  // a workgroup's items by groups and its rows by heads.
  int64_t block_tokens = R ? std::min<int64_t>(ROT_TOKENS, ROT_LDS_PAIRS / (R / 2)) : ROT_TOKENS;
  int64_t heads = p->HKV;
  const int64_t by_groups = (int64_t)a.groups * a.groups;
  auto held = [&] { return block_tokens * heads * std::max(by_groups, heads) < (1ll << 32); };
  while (block_tokens > 1 && (p->T / block_tokens < 1024 || !held())) block_tokens /= 2;
  while (!held()) heads = (heads + 1) / 2;
  a.block_tokens = (int32_t)block_tokens;
  a.block_heads = (int32_t)heads;
  a.groups_m = divider(a.groups);
  a.heads_m = divider(heads);
  a.magnitude = p->magnitude;
  hipStream_t s = (hipStream_t)stream;
  if (p->dtype == AFA_DTYPE_F16)
    return wide ? launch_append<DT_F16, 8>(a, p->layout, s) : launch_append<DT_F16, 1>(a, p->layout, s);
  return wide ? launch_append<DT_BF16, 8>(a, p->layout, s) : launch_append<DT_BF16, 1>(a, p->layout, s);
}
