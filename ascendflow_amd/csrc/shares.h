// What the attentions over a paged cache share, for gfx950: lengths of requests, the
// sums of a row and the split form, in which workgroups share the tiles of ragged
// requests evenly.
#pragma once

#include "common.h"

namespace afa {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// A tile of the split form as its merge needs it: its first row is row `row` of
// the packed rows of the request that starts at token `start`; workgroups
// first .. last hold parts of it (first == last: the tile is whole and written).
struct TileRecord {
  int32_t start, row, rows;
  int32_t first, last;
};

// Split form: the chunks of all tiles, in order, are one sequence that the
// workgroups share evenly, so that few or unequal requests fill the GPU and end
// together. A tile counts its chunks and 64 rows' worth for its start and end.
// Causal tiles of a request have unequal numbers of them: tiles i and n - 1 - i
// follow each other (the longer first) and count, together, what the first and
// the last tile do, so that any place in the sequence is found by a division.
// A workgroup takes at most one tile's end, whole tiles and one tile's
// beginning; parts go to the workspace (slot 2 w the end, 2 w + 1 the beginning)
// as float32 and latent_merge_kernel combines them in order. Everything is
// computed on the device from cu_seqlens_q and seqused_kv, alike in every workgroup.
//
// F, the form: ROWS (packed rows of a tile), KEYS (cache rows of a chunk), THREADS,
// START (chunks that a tile counts for its start and end), LEAST (chunks that a
// workgroup takes at least) and JOIN (below). A, the arguments of a kernel: cu, used,
// T, B, H (packed rows of a token), W, page_shift, causal, workers and tile_count.

// A row's ln(sum of e^scores) from its maximum m (log2) and its sum of weights:
// -inf for a sum of nothing. A sum that is not a number (scores that are none, or
// overflow to +inf) stays one, beside an output that is none either; it is told by its
// bits, since device code is built without NaN semantics of comparisons.
__device__ __forceinline__ float row_lse(float m, float total) {
  const uint32_t bits = __float_as_uint(total);
  uint32_t lse = __float_as_uint((m + __log2f(total)) * LN2);
  lse = (bits & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : lse;
  return __uint_as_float(bits == 0u ? 0xff800000u : lse);
}

// Metadata in the constant address space, so that uniform reads are scalar loads,
// whose values stay out of the vector registers and the vector load counter.
typedef const __attribute__((address_space(4))) int32_t* const_ints;
__device__ __forceinline__ const_ints constant(const int32_t* p) { return (const_ints)(uintptr_t)p; }

// New tokens of request b: cu[b] .. cu[b + 1], held inside [0, T).
__device__ __forceinline__ void request_tokens(const_ints cu, int b, int T, int& start, int& count) {
  start = min(max(cu[b], 0), T);
  count = max(min(cu[b + 1], T) - start, 0);
}

// Cache rows of request b that its table holds, and those ahead of its first new
// token (fewer than none where it has more tokens than rows). The tokens' places
// and so the causal limit go by the length itself, which may pass the table:
// token t sees rows up to ahead + t of the `used`.
template <typename A>
__device__ __forceinline__ void request_rows(const A& a, int b, int start, int& used, int& ahead) {
  const int length = max(constant(a.used)[b], 0);
  used = (int)min((int64_t)length, (int64_t)a.W << a.page_shift);
  ahead = length - (max(constant(a.cu)[b + 1], start) - start);
}

// The request and the tile inside it of tile `index` in the order of requests
// (tiles_of(tokens) each); false, for the whole workgroup, if there are fewer.
template <int THREADS, typename F>
__device__ __forceinline__ bool find_tile(const_ints cu, int B, int T, uint32_t index, F&& tiles_of, int& request,
                                          uint32_t& tile, uint32_t& tiles, uint32_t* words) {
  uint32_t* const wave_total = words;                // LDS, THREADS / 64 + 3 words
  uint32_t* const found = words + THREADS / 64;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  uint32_t before = 0;
  for (int base = 0; base < B; base += THREADS) {
    const int b = base + tid;
    int start = 0, count = 0;
    if (b < B) request_tokens(cu, b, T, start, count);
    const uint32_t mine = b < B ? tiles_of(count) : 0u;
    const uint32_t upto = (uint32_t)wave_inclusive_scan((int)mine);
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    uint32_t first = before, all = before;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) first += wave_total[w];
      all += wave_total[w];
    }
    const uint32_t begin = first + upto - mine;
    if (index >= begin && index < begin + mine) {
      found[0] = (uint32_t)b;
      found[1] = index - begin;
      found[2] = mine;
    }
    __syncthreads();
    if (index < all) {
      request = __builtin_amdgcn_readfirstlane((int)found[0]);
      tile = (uint32_t)__builtin_amdgcn_readfirstlane((int)found[1]);
      tiles = (uint32_t)__builtin_amdgcn_readfirstlane((int)found[2]);
      return true;
    }
    before = all;
  }
  return false;
}

// The part of the split form's sequence that a request takes.
template <typename F, typename A> struct TileSpan {
  static constexpr uint32_t ROWS = F::ROWS, START = F::START;
  int H, used, ahead, count, causal;
  uint32_t tiles;
  uint32_t pair, middle;  // what two paired tiles count, and the one left over
  __device__ __forceinline__ uint32_t chunks(uint32_t tile) const {
    const uint32_t last = min((tile + 1) * ROWS, (uint32_t)(count * H)) - 1;
    const int seen = causal ? min(max(ahead + (int)(last / (uint32_t)H) + 1, 0), used) : used;
    return ((uint32_t)seen + F::KEYS - 1) / F::KEYS;
  }
  __device__ __forceinline__ TileSpan(const A& a, int b) : H((int)opaque_uniform((uint32_t)a.H)), causal(a.causal) {
    int start;
    request_tokens(constant(a.cu), b, a.T, start, count);
    request_rows(a, b, start, used, ahead);
    tiles = ((uint32_t)(count * H) + ROWS - 1) / ROWS;
    const uint32_t most = ((uint32_t)used + F::KEYS - 1) / F::KEYS + START;
    pair = 2 * most;
    middle = most;
    if (causal && tiles > 1) {
      pair = most + chunks(0) + START;
      middle = chunks(tiles / 2) + START;
    }
  }
  __device__ __forceinline__ uint32_t longest() const {
    return tiles == 0 ? 0u : causal && tiles > 1 ? pair - chunks(0) - START : middle;
  }
  __device__ __forceinline__ uint64_t weight() const { return (uint64_t)(tiles / 2) * pair + (tiles % 2 ? middle : 0u); }
  // The tile at place `at` of the request's, and what it counts.
  __device__ __forceinline__ uint32_t tile(uint32_t at) const { return at % 2 || at + 1 == tiles ? at / 2 : tiles - 1 - at / 2; }
  __device__ __forceinline__ uint32_t longer(uint32_t p) const {
    return causal ? min(chunks(tiles - 1 - p) + START, pair - 1) : pair / 2;
  }
  __device__ __forceinline__ uint32_t counts(uint32_t at) const {
    if (at + 1 == tiles && tiles % 2) return middle;
    return at % 2 ? pair - longer(at / 2) : longer(at / 2);
  }
};

__device__ __forceinline__ uint64_t inclusive_scan64(uint64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t other = __shfl_up((unsigned long long)v, d);
    if (lane >= d) v += other;
  }
  return v;
}

// Maximum of the wave, in lane 63.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto with = [&](uint32_t other) { v = max(v, other); };
  with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr:1
  with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));  // row_shr:2
  with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));  // row_shr:4
  with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));  // row_shr:8
  with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return v;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
  return (uint64_t)(uint32_t)uniform((int)(uint32_t)v) | ((uint64_t)(uint32_t)uniform((int)(uint32_t)(v >> 32)) << 32);
}

// Sharing tiles costs the parts' bytes and the join, JOIN chunks' worth, and
// chunks take longer the more of the GPU is at work (3.2 us with half its CUs, 4.3
// with all: 128 rows of 512 columns are bound by power and by the L2s). Tiles are
// therefore kept whole where the longest of them, or the rounds that they need,
// take SHARE_APART times as many chunks as an even share and the join.
constexpr float SHARE_APART = 0.875f;

// Where a workgroup of the split form begins.
struct TileShare {
  uint64_t begin, end;       // of the sequence
  uint64_t total;
  int32_t workers;           // that have a share
  bool apart;                // tiles are not shared: a tile is whoever's its beginning is
  int32_t request;
  uint32_t place, offset;    // of the tile among the request's, inside the tile
  uint32_t tiles_before;     // of earlier requests
};

template <typename F, typename A>
__device__ __forceinline__ bool find_share(const A& a, uint32_t worker, uint32_t spread, TileShare& share) {
  constexpr int THREADS = F::THREADS;
  __shared__ uint64_t wave_weight[THREADS / 64];
  __shared__ uint32_t wave_tiles[THREADS / 64], wave_longest[THREADS / 64];
  __shared__ uint32_t found[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int per = (a.B + THREADS - 1) / THREADS;  // consecutive requests of a thread
  uint64_t weight = 0;
  uint32_t tiles = 0, longest = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b >= a.B) break;
    const TileSpan<F, A> span(a, b);
    weight += span.weight();
    tiles += span.tiles;
    longest = max(longest, span.longest());
  }
  const uint64_t upto = inclusive_scan64(weight, lane);
  const uint32_t tiles_upto = (uint32_t)wave_inclusive_scan((int)tiles);
  longest = wave_max(longest);
  if (lane == 63) {
    wave_weight[wave] = upto;
    wave_tiles[wave] = tiles_upto;
    wave_longest[wave] = longest;
  }
  __syncthreads();
  uint64_t before = upto - weight, total = 0;
  uint32_t tiles_before = tiles_upto - tiles, all = 0, most_chunks = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) {
      before += wave_weight[w];
      tiles_before += wave_tiles[w];
    }
    total += wave_weight[w];
    all += wave_tiles[w];
    most_chunks = max(most_chunks, wave_longest[w]);
  }
  total = uniform64(total);
  if (total == 0) {
    if (worker == 0 && tid == 0) *a.tile_count = 0;
    return false;
  }
  const uint64_t most = total / F::LEAST;
  share.workers = most < 1 ? 1 : (most < (uint64_t)a.workers ? (int)most : a.workers);
  share.workers = uniform(share.workers);
  all = (uint32_t)uniform((int)all);
  longest = (uint32_t)uniform((int)most_chunks);
  const float each = (float)total / (float)share.workers;
  const float whole = (float)((all + (uint32_t)share.workers - 1) / (uint32_t)share.workers) * ((float)total / (float)all);
  share.apart = __ballot(SHARE_APART * fmaxf((float)longest, whole) <= each + F::JOIN) != 0;
  const bool one = share.apart && all <= (uint32_t)a.workers;  // a tile each, spread over the XCDs
  worker = (uint32_t)uniform((int)(one ? spread : worker));
  if (worker >= (one ? all : (uint32_t)share.workers)) return false;
  if (worker == 0 && tid == 0) *a.tile_count = share.apart ? 0u : all;
  share.total = total;
  if (total < (1u << 22)) {  // 32-bit products with at most 512 workers: a 64-bit division costs microseconds
    share.begin = (uint32_t)uniform((int)((uint32_t)total * worker / (uint32_t)share.workers));
    share.end = (uint32_t)uniform((int)((uint32_t)total * (worker + 1) / (uint32_t)share.workers));
  } else {
    share.begin = uniform64(total * worker / (uint32_t)share.workers);
    share.end = uniform64(total * (worker + 1) / (uint32_t)share.workers);
  }
  if (one) {
    if (worker >= tiles_before && worker < tiles_before + tiles) {
      uint32_t place = worker - tiles_before;
      for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        const uint32_t mine = TileSpan<F, A>(a, b).tiles;
        if (place < mine) {
          found[0] = (uint32_t)b;
          found[1] = place;
          found[2] = 0;
          found[3] = 0;
          break;
        }
        place -= mine;
      }
    }
  } else if (share.begin >= before && share.begin < before + weight) {
    uint64_t at = before;
    uint32_t done = tiles_before;
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      const TileSpan<F, A> span(a, b);
      if (share.begin < at + span.weight()) {
        const uint64_t inside = share.begin - at;
        const uint32_t pairs = (uint32_t)min(inside / span.pair, (uint64_t)(span.tiles / 2));
        uint32_t offset = (uint32_t)(inside - (uint64_t)pairs * span.pair), place = 2 * pairs;
        if (pairs < span.tiles / 2) {
          const uint32_t longer = span.longer(pairs);
          if (offset >= longer) {
            offset -= longer;
            ++place;
          }
        }
        found[0] = (uint32_t)b;
        found[1] = place;
        found[2] = offset;
        found[3] = done;
        break;
      }
      at += span.weight();
      done += span.tiles;
    }
  }
  __syncthreads();
  if (one) share.end = share.begin + 1;
  share.request = uniform((int)found[0]);
  share.place = (uint32_t)uniform((int)found[1]);
  share.offset = (uint32_t)uniform((int)found[2]);
  share.tiles_before = (uint32_t)uniform((int)found[3]);
  return true;
}

}  // namespace afa
