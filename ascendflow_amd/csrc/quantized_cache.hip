// Append of new tokens to a paged cache held in 8 bits, for gfx950.
//
// A block of GROUP tokens of one head shares a scale s: the codes c of its keys (and,
// with a scale of their own, of its values) stand for c s. With A the largest finite
// magnitude of a block's new rows and C the largest code (448 for e4m3, 127 for int8),
//   need = 2^max(ceil(log2(A / C)), -80),   s = max(need, s of the rows it held before),
//   c = round(x / s), to nearest, ties to even, held inside [-C, C],
// and rows that the block held before are rounded anew where s grew. A power of two
// wastes at most one bit of int8's range and none of e4m3's precision, and makes the
// rounding anew exact (e4m3, but for codes that fall among its subnormals) or a shift
// with a rounding (int8), which leaves a code within one step of the last scale however the
// block was filled. The exponent comes from the bits of A, so nothing is rounded but x / s.
//
// One wave takes the new rows of one block, of one head's keys or values: a pass for A,
// the rows held before where the scale grows, a pass for the codes, the rows in registers
// between them (3 prompts of 1000 to 1987 tokens, 8 heads of 128 int8 columns 13.7 -> 10.0
// us, with codes in 3 operations a value where all are finite instead of 13). Bound by HBM
// where tokens are many, else by the launch and a chain of dependent loads (lengths, table,
// scale; the rows' own are under way beside it): 64 decode tokens of 8 heads 4.8 us.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "../../include/ascendflow_amd.h"

namespace afa {

constexpr int Q8_LEAST = -80;      // exponent of the least scale
constexpr int Q8_MAX_D = 1024, Q8_MAX_GROUP = 1024, Q8_MAX_HKV = 32768;

struct AppendQuantizedArgs {
  const void* x[2];       // keys, values
  uint8_t* cache[2];
  float* scale[2];
  const int32_t* table;
  const int32_t* cu;
  const int32_t* used;
  int64_t x_t[2], x_h[2];
  int32_t T, B, W, page_shift, group_shift, BLOCKS, HKV, D;
  uint32_t pieces_m;      // divides by the pieces of a row
};

// index / n for index * n < 2^32, with m = ceil(2^32 / n) (0 for n = 1).
__device__ __forceinline__ uint32_t q8_divide(uint32_t index, uint32_t m) { return m ? __umulhi(index, m) : index; }

__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

// The least power of two, from 2^Q8_LEAST on, that holds magnitudes up to `top` (finite, by its bits).
template <int CT>
__device__ __forceinline__ float needed_scale(uint32_t top) {
  const int limit = CT == AFA_CODE_E4M3 ? 0x600000 : 0x7e0000;  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const int least_bits = CT == AFA_CODE_E4M3 ? 8 : 6;
  const int exponent = (int)(top >> 23) - 127 - least_bits + ((int)(top & 0x7fffffu) > limit ? 1 : 0);
  return __uint_as_float((uint32_t)(max(exponent, Q8_LEAST) + 127) << 23);
}

// Two codes from values in units of their scale, in the low 16 bits.
template <int CT>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  constexpr float C = CT == AFA_CODE_E4M3 ? 448.0f : 127.0f;
  // Comparisons that a NaN fails leave it: e4m3 has a code for it, int8 takes 0.
  a = a > C ? C : (a < -C ? -C : a);
  b = b > C ? C : (b < -C ? -C : b);
  if constexpr (CT == AFA_CODE_E4M3) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
  } else {
    a = a == a ? a : 0.0f;
    b = b == b ? b : 0.0f;
    return ((uint32_t)(int)__builtin_rintf(a) & 0xffu) | (((uint32_t)(int)__builtin_rintf(b) & 0xffu) << 8);
  }
}

// Four codes from values that round to codes. int8: next to 1.5 * 2^23 a float32 keeps whole numbers, in its low bits.
template <int CT>
__device__ __forceinline__ uint32_t encode4(const float* v) {
#pragma clang fp contract(off)
  if constexpr (CT == AFA_CODE_E4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
  } else {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(v[i] + 12582912.0f);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
  }
}

template <int CT>
__device__ __forceinline__ float decode1(uint32_t code) {
  if constexpr (CT == AFA_CODE_E4M3)
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
  else
    return (float)(int8_t)code;
}

template <int DT, int VEC> struct Piece16 { typedef typename B16<DT>::x8 type; };
template <int DT> struct Piece16<DT, 1> { typedef typename B16<DT>::scalar type __attribute__((ext_vector_type(1))); };

// VEC columns of a row: 8 (16 bytes of new values, 8 of codes) or 1.
template <int DT, int CT, int VEC>
__global__ __launch_bounds__(256) void append_quantized_kernel(AppendQuantizedArgs a) {
#pragma clang fp contract(off)  // x / s is rounded before it becomes a code
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x8 x8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.y * 4u + (uint32_t)wave;
  const int which = (int)(item & 1u), head = (int)(item >> 1);
  if (head >= a.HKV) return;

  // The block: each request's new tokens touch a run of blocks; this wave's is number blockIdx.x of them all.
  int request = -1, first = 0, count = 0, limit = 0, block = 0;
  {
    uint32_t before = 0;
    const uint32_t index = blockIdx.x;
    for (int base = 0; base < a.B; base += 64) {
      const int b = base + lane;
      int start = 0, n = 0, low = 0, high = 0, stop = 0;
      uint32_t mine = 0;
      if (b < a.B) {
        stop = a.cu[b + 1];
        start = min(max(a.cu[b], 0), a.T);
        n = max(min(stop, a.T) - start, 0);
        // Token t lies at used - cu[b + 1] + t; positions below 0 or past the table are not there.
        const int64_t place = (int64_t)a.used[b] - stop + start;
        const int64_t held = (int64_t)a.W << a.page_shift;
        low = (int)min(max(place, (int64_t)0), held);
        high = (int)min(max(place + n, (int64_t)0), held);
        if (high > low) mine = (uint32_t)(((high - 1) >> a.group_shift) - (low >> a.group_shift) + 1);
        start = (int)(low - place) + start;  // the token at position `low`
      }
      const uint32_t upto = (uint32_t)wave_inclusive_scan((int)mine) + before;
      const uint64_t has = __ballot(mine > 0 && index >= upto - mine && index < upto);
      if (has) {
        const int l = __ffsll((unsigned long long)has) - 1;
        request = base + l;
        first = __builtin_amdgcn_readlane(low, l);
        limit = __builtin_amdgcn_readlane(high, l);
        count = __builtin_amdgcn_readlane(start, l);
        block = (first >> a.group_shift) + (int)(index - (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), l));
        break;
      }
      before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
  }
  if (request < 0) return;
  const int G = 1 << a.group_shift;
  const int at = block << a.group_shift;              // position of the block's first row
  const int low = max(first, at), high = min(limit, at + G);
  const int64_t token = (int64_t)count + (low - first);  // at position `low`
  const int pieces = a.D / VEC, held = low - at, rows = high - low;
  const scalar* const x = (const scalar*)a.x[which] + token * a.x_t[which] + head * a.x_h[which];
  // The new rows, KEEP pieces of which stay in registers between the two passes: every one of 64 rows of 128 columns.
  constexpr int KEEP = VEC == 8 ? 16 : 8;
  typedef typename Piece16<DT, VEC>::type piece;
  const uint32_t n = (uint32_t)(rows * pieces);
  auto new_piece = [&](uint32_t i) {
    const uint32_t r = q8_divide(i, a.pieces_m), c = i - r * (uint32_t)pieces;
    return *(const piece*)(x + r * a.x_t[which] + c * VEC);
  };
  piece kept[KEEP];
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const uint32_t i = lane + 64u * k;
    if (64u * k < n) kept[k] = new_piece(min(i, n - 1));  // a piece again where there is none: the same largest magnitude
  }
  // Under way before the page is known.
  const int page = a.table[(int64_t)request * a.W + (at >> a.page_shift)];
  if (page < 0 || page >= a.BLOCKS) return;
  const int64_t row0 = ((int64_t)page << a.page_shift) + (at & ((1 << a.page_shift) - 1));
  float* const scale_at = a.scale[which] + (row0 >> a.group_shift) * a.HKV + head;
  const int64_t row_stride = (int64_t)a.HKV * a.D;
  uint8_t* const codes = a.cache[which] + (row0 * a.HKV + head) * a.D;
  const float had = held > 0 ? *scale_at : 0.0f;

  // The largest magnitude: of 16-bit values two at a time, where it is finite, else one by one.
  uint32_t top = 0;
  bool finite = false;
  if constexpr (VEC == 8) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0};
    auto largest2 = [&](const piece& p) {
      const u32x4 w = __builtin_bit_cast(u32x4, p);
#pragma unroll
      for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
    };
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (64u * k < n) largest2(kept[k]);
    for (uint32_t i = lane + 64u * KEEP; i < n; i += 64) largest2(new_piece(i));
    const uint32_t bits = wave_max_bits(max((uint32_t)most[0], (uint32_t)most[1]));
    finite = __builtin_amdgcn_readfirstlane((int)bits) < (DT == DT_BF16 ? 0x7f80 : 0x7c00);
    top = __float_as_uint((float)__builtin_bit_cast(scalar, (uint16_t)bits));
  }
  if (!finite) top = 0;
  auto largest = [&](const piece& p) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t bits = __float_as_uint((float)p[e]) & 0x7fffffffu;
      top = max(top, bits < 0x7f800000u ? bits : 0u);
    }
  };
  if (!finite) {
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (64u * k < n) largest(kept[k]);
    for (uint32_t i = lane + 64u * KEEP; i < n; i += 64) largest(new_piece(i));
    top = wave_max_bits(top);
  }
  float now = needed_scale<CT>(top);
  if (held > 0) now = now > had ? now : (had == had ? had : now);
  const float inverse = 1.0f / now;

  auto put = [&](uint8_t* to, const float* v) {
    if constexpr (VEC == 8) {
      u32x2 w;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h] = encode2<CT>(v[4 * h], v[4 * h + 1]) | (encode2<CT>(v[4 * h + 2], v[4 * h + 3]) << 16);
      *(u32x2*)to = w;
    } else {
      *to = (uint8_t)encode2<CT>(v[0], 0.0f);
    }
  };
  if (held > 0 && now != had) {
    for (uint32_t i = lane; i < (uint32_t)(held * pieces); i += 64) {
      const uint32_t r = q8_divide(i, a.pieces_m), c = i - r * (uint32_t)pieces;
      uint8_t* p = codes + r * row_stride + c * VEC;
      float v[VEC];
      if constexpr (VEC == 8) {
        const u32x2 w = *(const u32x2*)p;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = decode1<CT>((w[e / 4] >> (8 * (e % 4))) & 0xffu) * had * inverse;
      } else {
        v[0] = decode1<CT>(*p) * had * inverse;
      }
      put(p, v);
    }
  }
  auto put_new = [&](uint32_t i, const piece& p) {
    const uint32_t r = q8_divide(i, a.pieces_m), c = i - r * (uint32_t)pieces;
    uint8_t* const to = codes + (held + (int)r) * row_stride + c * VEC;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)p[e] * inverse;
    if (VEC == 8 && finite) {  // nothing to hold inside the range: the scale holds the largest magnitude
      u32x2 w;
#pragma unroll
      for (int h = 0; h < 2; ++h) w[h] = encode4<CT>(v + 4 * h);
      *(u32x2*)to = w;
    } else {
      put(to, v);
    }
  };
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (lane + 64u * k < n) put_new(lane + 64u * k, kept[k]);
  for (uint32_t i = lane + 64u * KEEP; i < n; i += 64) put_new(i, new_piece(i));
  if (lane == 0) *scale_at = now;
}

namespace {

bool q8_on(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int shift_of(int32_t power) {
  int s = 0;
  while ((1 << s) < power) ++s;
  return s;
}

template <int DT, int CT>
int launch_append_as(const AppendQuantizedArgs& a, bool wide, hipStream_t s) {
  const int64_t G = 1ll << a.group_shift;
  const int64_t blocks = std::min<int64_t>(a.T, a.T / G + 2ll * a.B);  // n tokens touch at most min(n, (n - 2) / G + 2)
  const dim3 grid((unsigned)blocks, (unsigned)((2 * a.HKV + 3) / 4)), block(256);
  if (wide)
    hipLaunchKernelGGL((append_quantized_kernel<DT, CT, 8>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((append_quantized_kernel<DT, CT, 1>), grid, block, 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace afa

extern "C" int launch_append_quantized_kv(void* stream, const void* k, const void* v, const int32_t* block_table,
                                          const int32_t* cu_seqlens_q, const int32_t* seqused_kv, void* k_cache,
                                          void* v_cache, float* k_scale, float* v_scale,
                                          const AppendQuantizedKvParams* p) {
  using namespace afa;
  if (!p) return AFA_E_NULL;
  if ((p->dtype != AFA_DTYPE_BF16 && p->dtype != AFA_DTYPE_F16) || (p->code != AFA_CODE_E4M3 && p->code != AFA_CODE_INT8))
    return AFA_E_DTYPE;
  if (p->T < 0 || p->B <= 0 || p->W <= 0 || p->BLOCKS <= 0 || p->HKV <= 0 || p->D <= 0) return AFA_E_SHAPE;
  if (p->D > Q8_MAX_D || p->HKV > Q8_MAX_HKV || p->GROUP > Q8_MAX_GROUP || p->T >= 1 << 23 || p->B >= 1 << 23) return AFA_E_SHAPE;
  if (p->GROUP < 16 || (p->GROUP & (p->GROUP - 1)) || p->PAGE < p->GROUP || (p->PAGE & (p->PAGE - 1))) return AFA_E_SHAPE;
  if ((int64_t)p->W * p->PAGE > 1ll << 30) return AFA_E_SHAPE;  // positions are 32-bit numbers
  if (!k || !v || !block_table || !cu_seqlens_q || !seqused_kv || !k_cache || !v_cache || !k_scale || !v_scale)
    return AFA_E_NULL;
  if (p->T == 0) return AFA_OK;
  AppendQuantizedArgs a;
  a.x[0] = k;
  a.x[1] = v;
  a.cache[0] = (uint8_t*)k_cache;
  a.cache[1] = (uint8_t*)v_cache;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.table = block_table;
  a.cu = cu_seqlens_q;
  a.used = seqused_kv;
  a.x_t[0] = p->k_stride_t;
  a.x_h[0] = p->k_stride_h;
  a.x_t[1] = p->v_stride_t;
  a.x_h[1] = p->v_stride_h;
  a.T = p->T;
  a.B = p->B;
  a.W = p->W;
  a.page_shift = shift_of(p->PAGE);
  a.group_shift = shift_of(p->GROUP);
  a.BLOCKS = p->BLOCKS;
  a.HKV = p->HKV;
  a.D = p->D;
  const bool wide = p->D % 8 == 0 && q8_on(k, 16) && q8_on(v, 16) && q8_on(k_cache, 8) && q8_on(v_cache, 8) &&
                    (p->k_stride_t | p->k_stride_h | p->v_stride_t | p->v_stride_h) % 8 == 0;
  const int64_t pieces = wide ? p->D / 8 : p->D;
  a.pieces_m = pieces == 1 ? 0u : (uint32_t)(((1ull << 32) + pieces - 1) / pieces);
  hipStream_t s = (hipStream_t)stream;
  const bool f16 = p->dtype == AFA_DTYPE_F16;
  if (p->code == AFA_CODE_E4M3)
    return f16 ? launch_append_as<DT_F16, AFA_CODE_E4M3>(a, wide, s) : launch_append_as<DT_BF16, AFA_CODE_E4M3>(a, wide, s);
  return f16 ? launch_append_as<DT_F16, AFA_CODE_INT8>(a, wide, s) : launch_append_as<DT_BF16, AFA_CODE_INT8>(a, wide, s);
}
