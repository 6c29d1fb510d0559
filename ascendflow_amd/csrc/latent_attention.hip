// Attention whose keys and values come from one latent vector a token, for
// gfx950: the absorbed form over a paged cache and the expanded form over
// contiguous keys and values.
//
// Absorbed (latent_attention): a cache row is [c | k_rope], c of L columns, one
// row for all heads. With the key projection absorbed into the query,
//   s = scale (q . c + q_rope . k_rope),  o = softmax(s) c,
// so a row is read once and serves as key and as value. The rows of a request's
// (token, head) pairs are packed token by token into tiles of 16 * NW rows; each
// wave owns 16 of them, whose Q (L + R columns) and O (L columns, float32) stay
// in registers. Cache rows stream in chunks of 64 or 32 through an LDS ring filled by
// the load-to-LDS path, XOR-swizzled on the global side, and every wave reads
// every row twice: S^T[keys, rows] = K Q^T with ds_read_b128, O^T[columns, rows]
// += V^T P^T with the transposing ds_read_b64_tr_b16. P stays in the wave's
// registers (the accumulator layout of S^T is the operand layout of P^T, up to
// an order of keys that both sides share), so a chunk costs one barrier.
//
// Online softmax in float32, exp2 domain: the running maximum m is raised when a
// row's maximum exceeds it by more than lat_tau (log2 units): 8 with float16, so
// that O is rescaled rarely, 0 with bfloat16. P <= 2^lat_tau is rounded to the
// storage type (a matrix operand has to be), at most half a step of each weight,
// while O is divided by the sum of the weights before rounding. Of a row that one
// key dominates that key's own rounding is the error: none where it holds the
// maximum (its weight is 1), up to half a step where the maximum lags, 2^-11 in
// float16 but 2^-8 in bfloat16. (Raising it at any growth costs 5% of 8192 causal
// tokens of 32 heads, expanded, 604 -> 633 us, and 0 to 3% of the absorbed calls.
// The sum of the rounded weights would cancel that error too, but costs a
// conversion and an addition a score: 700 us.)
#include <algorithm>
#include <cmath>

#include "common.h"
#include "../../include/ascendflow_amd.h"

namespace afa {

constexpr float LAT_LOG2E = 1.4426950408889634f, LAT_LN2 = 0.6931471805599453f;
template <int DT> __device__ constexpr float lat_tau() { return DT == DT_F16 ? 8.0f : 0.0f; }
constexpr int EXP_MAX_SPLITS = 64;
// Cache rows per chunk. Eight waves (one workgroup per CU): 64, two slots; a
// barrier, a fetch and a reduction per 64 rows instead of 32 and four chains of
// dependent matrix instructions instead of two (128 heads, 4 chunks of 512 tokens
// behind 8K: 4317 -> 3865 us when it was taken). Four waves: 32, two slots in each of the CU's two
// workgroups.
template <int NW> __host__ __device__ constexpr int lat_keys() { return NW == 8 ? 64 : 32; }

struct LatentArgs {
  const void* q;
  const void* q_rope;
  const void* cache;
  const int32_t* table;
  const int32_t* cu;
  const int32_t* used;
  void* out;
  float* lse;  // [T][H] or NULL
  int64_t q_t, q_h, qr_t, qr_h, o_t, o_h;
  int32_t T, B, H, W, page_shift, blocks, causal;
  float scale;
  // Split form (below): workgroups, and its workspace.
  int32_t workers;
  float* partial_o;         // [2 * workers][rows of a tile / 16][L / 16][64][4], not normalised, as a wave holds it
  float* partial_ml;        // [2 * workers][rows of a tile][2]: running maximum (log2), sum of weights
  struct LatentRecord* records;  // [tiles]
  uint32_t* tile_count;
  uint32_t tiles;           // the most that monotone cu_seqlens_q can give
};

// A tile of the split form as its merge needs it: its first row is row `row` of
// the packed rows of the request that starts at token `start`; workgroups
// first .. last hold parts of it (first == last: the tile is whole and written).
struct LatentRecord {
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
template <int NW> __host__ __device__ constexpr uint32_t lat_start() { return 64 / lat_keys<NW>(); }
template <int NW> __host__ __device__ constexpr uint32_t lat_least() { return 128 / lat_keys<NW>(); }  // least of a workgroup

// A row's ln(sum of e^scores) from its maximum m (log2) and its sum of weights:
// -inf for a sum of nothing. A sum that is not a number (scores that are none, or
// overflow to +inf) stays one, beside an output that is none either; it is told by its
// bits, since device code is built without NaN semantics of comparisons.
__device__ __forceinline__ float row_lse(float m, float total) {
  const uint32_t bits = __float_as_uint(total);
  uint32_t lse = __float_as_uint((m + __log2f(total)) * LAT_LN2);
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
__device__ __forceinline__ void request_rows(const LatentArgs& a, int b, int start, int& used, int& ahead) {
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
template <int NW> struct LatentSpan {
  static constexpr uint32_t ROWS = 16 * NW, START = lat_start<NW>();
  int H, used, ahead, count, causal;
  uint32_t tiles;
  uint32_t pair, middle;  // what two paired tiles count, and the one left over
  __device__ __forceinline__ uint32_t chunks(uint32_t tile) const {
    const uint32_t last = min((tile + 1) * ROWS, (uint32_t)(count * H)) - 1;
    const int seen = causal ? min(max(ahead + (int)(last / (uint32_t)H) + 1, 0), used) : used;
    return ((uint32_t)seen + lat_keys<NW>() - 1) / lat_keys<NW>();
  }
  __device__ __forceinline__ LatentSpan(const LatentArgs& a, int b) : H((int)opaque_uniform((uint32_t)a.H)), causal(a.causal) {
    int start;
    request_tokens(constant(a.cu), b, a.T, start, count);
    request_rows(a, b, start, used, ahead);
    tiles = ((uint32_t)(count * H) + ROWS - 1) / ROWS;
    const uint32_t most = ((uint32_t)used + lat_keys<NW>() - 1) / lat_keys<NW>() + START;
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

// Sharing tiles costs the parts' bytes and the join, LAT_JOIN chunks' worth, and
// chunks take longer the more of the GPU is at work (3.2 us with half its CUs, 4.3
// with all: 128 rows of 512 columns are bound by power and by the L2s). Tiles are
// therefore kept whole where the longest of them, or the rounds that they need,
// take LAT_APART times as many chunks as an even share and the join.
constexpr float LAT_APART = 0.875f;
template <int NW> constexpr float LAT_JOIN = NW == 8 ? 5.0f : 10.0f;

// Where a workgroup of the split form begins.
struct LatentShare {
  uint64_t begin, end;       // of the sequence
  uint64_t total;
  int32_t workers;           // that have a share
  bool apart;                // tiles are not shared: a tile is whoever's its beginning is
  int32_t request;
  uint32_t place, offset;    // of the tile among the request's, inside the tile
  uint32_t tiles_before;     // of earlier requests
};

template <int NW>
__device__ __forceinline__ bool find_share(const LatentArgs& a, uint32_t worker, LatentShare& share) {
  constexpr int THREADS = NW * 64;
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
    const LatentSpan<NW> span(a, b);
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
  const uint64_t most = total / lat_least<NW>();
  share.workers = most < 1 ? 1 : (most < (uint64_t)a.workers ? (int)most : a.workers);
  share.workers = uniform(share.workers);
  all = (uint32_t)uniform((int)all);
  longest = (uint32_t)uniform((int)most_chunks);
  const float each = (float)total / (float)share.workers;
  const float whole = (float)((all + (uint32_t)share.workers - 1) / (uint32_t)share.workers) * ((float)total / (float)all);
  share.apart = __ballot(LAT_APART * fmaxf((float)longest, whole) <= each + LAT_JOIN<NW>) != 0;
  const bool one = share.apart && all <= (uint32_t)a.workers;  // a tile each, spread over the XCDs
  worker = (uint32_t)uniform((int)(one ? blockIdx.x : worker));
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
        const uint32_t mine = LatentSpan<NW>(a, b).tiles;
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
      const LatentSpan<NW> span(a, b);
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

// STREAM: non-temporal loads, for requests of one tile each (nothing is read
// twice) over a cache too large to stay in the 256 MiB Infinity Cache between
// calls (64 requests of 32K with 128 heads 627 -> 616 us, 32 with 16 heads 222 -> 200;
// 64 of 2K with 16 heads, 150 MB, 43.6 -> 43.9).
template <int DT, int L, int R, int NW, bool SPLIT, bool STREAM>
__global__ __launch_bounds__(NW * 64, NW == 8 ? 1 : 2) void latent_kernel(LatentArgs a) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x8 x8;
  typedef typename B16<DT>::x4 x4;
  static_assert(L % 128 == 0 && L <= 512 && (R == 0 || R == 64) && (NW == 4 || NW == 8), "supported rows");
  constexpr int ROWS = 16 * NW;
  constexpr int LROW = 2 * L;                  // bytes of a latent row in LDS
  constexpr int GROW = 2 * (L + R);            // bytes of a cache row
  constexpr int KEYS = lat_keys<NW>(), KT = KEYS / 16;
  constexpr int ROPE_AT = KEYS * LROW;         // the rotary parts follow the latents
  constexpr int SLOT = KEYS * GROW;
  constexpr int NS = NW == 8 && L < 512 ? 3 : 2;  // ring slots: what 160 KiB hold for one workgroup per CU, or two
  constexpr int RW = 8;                        // rows that one wave loads
  static_assert(RW * NW == KEYS, "a chunk is loaded by all waves");
  constexpr int LR = 512 / L, LOADS_L = RW / LR, LOADS = LOADS_L + (R ? 1 : 0);
  constexpr int KSTEPS = L / 32, RSTEPS = R / 32, VTILES = L / 16;
  __shared__ __attribute__((aligned(256))) uint8_t ring[NS][SLOT];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, i16 = lane & 15;
  const int H = a.H;
  // Parts of one tile, and tiles of one request, on one XCD (they share its L2).
  const uint32_t worker = SPLIT ? xcd_contiguous(blockIdx.x, gridDim.x) : blockIdx.x;

  int request;
  uint32_t tile, tiles;
  uint32_t place = 0;  // of the tile among its request's in the split form's order
  LatentShare share;
  uint64_t left = 0;   // of this workgroup's share
  if constexpr (SPLIT) {
    if (!find_share<NW>(a, worker, share)) return;
    request = share.request;
    place = share.place;
    left = share.end - share.begin;
  } else {
    if (!find_tile<NW * 64>(constant(a.cu), a.B, a.T, worker,
                            [&](int n) { return ((uint32_t)n * (uint32_t)H + ROWS - 1) / ROWS; }, request, tile, tiles,
                            (uint32_t*)ring[0]))
      return;
    __syncthreads();  // the words are read before loads land on them
    if (a.causal) tile = tiles - 1 - tile;  // the longest first
  }
  uint32_t offset = SPLIT ? share.offset : 0;
  const float scale_log2 = a.scale * LAT_LOG2E;

  for (bool first_part = true;; first_part = false) {
  if (SPLIT && request >= a.B) return;  // never, unless cu_seqlens_q or seqused_kv change under the call
  int start, count;
  request_tokens(constant(a.cu), request, a.T, start, count);
  int used, ahead;
  request_rows(a, request, start, used, ahead);
  const int rows = count * H;
  uint32_t each = 0;  // what the tile counts
  if constexpr (SPLIT) {
    const LatentSpan<NW> span(a, request);
    if (place >= span.tiles) {  // on to the next request that has tokens (there is one: something is left)
      share.tiles_before += span.tiles;
      place = 0;
      ++request;
      continue;
    }
    tile = (uint32_t)uniform((int)span.tile(place));
    each = (uint32_t)uniform((int)span.counts(place));
    if (share.apart && offset > 0) {  // an earlier workgroup's tile
      if (left <= each - offset) return;
      left -= each - offset;
      offset = 0;
      ++place;
      continue;
    }
  }

  auto visible = [&](int t) { return a.causal ? min(max(ahead + t + 1, 0), used) : used; };
  // This lane's (token, head) row. Worked out where it is needed (Q, masks, the
  // end): kept, it would cost registers that the loop does not have.
  auto my_row = [&](int& token, int& head) {
    const int row = (int)(tile * ROWS) + (int)(opaque((uint32_t)tid) >> 6) * 16 + (int)(opaque((uint32_t)tid) & 15u);
    token = row < rows ? row / H : 0;
    head = row - token * H;
    return row < rows;
  };
  const int kv_end = visible((min((int)(tile + 1) * ROWS, rows) - 1) / H);
  const int clean_end = visible((int)tile * ROWS / H);  // no row of the tile hides a key below
  // This wave has no rows: it only loads (the direct form, whose tiles are nearly all full, spills with the branch).
  const bool idle = SPLIT && (int)(tile * ROWS) + wave * 16 >= rows;
  const int all_chunks = (kv_end + KEYS - 1) / KEYS;
  int begin = 0, chunks = all_chunks;  // of this part
  bool whole = true;
  if constexpr (SPLIT) {
    // The tile's own chunks, spread over what it counts.
    constexpr uint32_t START = lat_start<NW>();
    const uint32_t end = share.apart ? each : (uint32_t)min((uint64_t)each, (uint64_t)offset + left);
    auto cut = [&](uint32_t x) {
      return x >= each ? all_chunks : (x <= START ? 0 : (int)((uint64_t)(x - START) * (uint32_t)all_chunks / (each - START)));
    };
    begin = cut(offset);
    chunks = cut(end);
    whole = offset == 0 && end == each;
    if (!share.apart && offset == 0 && tid == 0 && share.tiles_before + place < a.tiles) {
      const uint64_t tile_end = share.end - left + each;  // in the sequence
      LatentRecord r;
      r.start = start;
      r.row = (int)tile * ROWS;
      r.rows = min(ROWS, rows - (int)tile * ROWS);
      r.first = (int)worker;
      // Divisions from scratch: their divisors' reciprocals, kept, would be spilled.
      const uint32_t low = opaque_uniform((uint32_t)share.total), high = opaque_uniform((uint32_t)(share.total >> 32));
      r.last = share.total < (1u << 22) ? (int)(((uint32_t)tile_end * (uint32_t)share.workers - 1) / low)
                                        : (int)((tile_end * (uint32_t)share.workers - 1) / ((uint64_t)high << 32 | low));
      a.records[share.tiles_before + place] = r;
    }
    left -= min(left, (uint64_t)(end - offset));
    if (!first_part) block_barrier();  // the ring is read
  }

  // ---- cache rows to LDS -----------------------------------------------------
  const uint32_t ring_base = lds_address(ring[0]);
  const const_ints pages = constant(a.table + (int64_t)request * a.W);
  const int page_mask = (1 << a.page_shift) - 1;
  auto inside = [&](int page) { return (uint32_t)page < (uint32_t)a.blocks; };
  int page[KT];        // of the 16-row groups of the next chunk to load, -1 past the end
  uint32_t good = 0;   // KT bits per chunk loaded, the latest lowest: its groups' pages lie in the cache
  int partial = 0;     // chunks until every one in flight has all its loads
  auto look_up = [&](int chunk) {
    const int key = chunk * KEYS;
    if (a.page_shift >= (KEYS == 64 ? 6 : 5)) {  // one page
      page[0] = key < kv_end ? pages[key >> a.page_shift] : -1;
#pragma unroll
      for (int i = 1; i < KT; ++i) page[i] = key + 16 * i < kv_end ? page[0] : -1;
    } else {
#pragma unroll
      for (int i = 0; i < KT; ++i) page[i] = key + 16 * i < kv_end ? pages[(key + 16 * i) >> a.page_shift] : -1;
    }
  };
  auto fetch = [&](int chunk) {
    const int first = wave * RW, group = first >> 4;  // of the chunk's rows
    const int key = chunk * KEYS + first;
    int mine = page[0];
    uint32_t bits = inside(page[0]) ? 1u : 0u;
#pragma unroll
    for (int i = 1; i < KT; ++i) {
      bits |= inside(page[i]) ? 1u << i : 0u;
      mine = group == i ? page[i] : mine;
    }
    good = (good << KT) | bits;
    const int have = (bits >> group) & 1u ? min(max(kv_end - key, 0), RW) : 0;
    const char* from = (const char*)a.cache + (((int64_t)mine << a.page_shift) + (key & page_mask)) * GROW;
    const uint32_t slot = ring_base + (uint32_t)((chunk - begin) % NS) * SLOT;
    const uint32_t to = opaque_uniform(slot + (uint32_t)(first * LROW));
    const uint32_t to_rope = opaque_uniform(slot + (uint32_t)(ROPE_AT + first * 2 * R));
    if (partial > 0) --partial;
    if (have < RW) partial = NS;
    const uint32_t ln = opaque((uint32_t)tid) & 63u;  // offsets worked out anew: kept, they would be spilled
    auto load = [&](uint32_t dst, uint32_t off) {
      if constexpr (STREAM)
        __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                         :: "s"(dst), "v"(off), "s"(from) : "memory");
      else
        __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                         :: "s"(dst), "v"(off), "s"(from) : "memory");
    };
    const int r0 = (int)(ln / (L / 8)), rope_row = (int)(ln >> 3);
    auto latent_off = [&](int r) {
      return (uint32_t)(r * GROW) + (((ln % (L / 8)) ^ (uint32_t)((first + r) & 15)) << 4);
    };
    auto rope_off = [&]() {
      return (uint32_t)(rope_row * GROW + LROW) + (((ln & 7u) ^ (uint32_t)(((first + rope_row) >> 1) & 7)) << 4);
    };
    if (have == RW) {
#pragma unroll
      for (int p = 0; p < LOADS_L; ++p) load(to + (uint32_t)p * 1024u, latent_off(p * LR + r0));
      if constexpr (R != 0)
        load(to_rope, rope_off());
    } else {
      // Rows past the end or without a page become zeros, which no weight can turn into anything else.
      const uint32_t none = opaque(0u);  // not a register kept through the loop
      const u32x4 zero = {none, none, none, none};
#pragma unroll
      for (int p = 0; p < LOADS_L; ++p) {
        if (p * LR + r0 < have)
          load(to + (uint32_t)p * 1024u, latent_off(p * LR + r0));
        else
          *(AFA_LDS u32x4*)(uintptr_t)(to + (uint32_t)p * 1024u + ln * 16u) = zero;
      }
      if constexpr (R != 0) {
        if (rope_row < have)
          load(to_rope, rope_off());
        else
          *(AFA_LDS u32x4*)(uintptr_t)(to_rope + ln * 16u) = zero;
      }
    }
  };

  // ---- Q fragments: B operand, columns 32 j + 8 g .. + 7 of row i16 -----------
  x8 qf[KSTEPS + RSTEPS];
  {
    int token, head;
    const bool valid = my_row(token, head);
    if (!valid) head = 0;
    const scalar* q = (const scalar*)a.q + (int64_t)(start + token) * a.q_t + (int64_t)head * a.q_h + 8 * g;
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j)
      qf[j] = valid ? *(const x8*)(q + 32 * j) : __builtin_bit_cast(x8, u32x4{0u, 0u, 0u, 0u});
    if constexpr (R != 0) {
      const scalar* qr = (const scalar*)a.q_rope + (int64_t)(start + token) * a.qr_t + (int64_t)head * a.qr_h + 8 * g;
#pragma unroll
      for (int j = 0; j < RSTEPS; ++j)
        qf[KSTEPS + j] = valid ? *(const x8*)(qr + 32 * j) : __builtin_bit_cast(x8, u32x4{0u, 0u, 0u, 0u});
    }
  }

  // ---- fragment addresses (relative to a slot; XOR picks the 64- or 32-byte group) --
  const int ra = sigma(i16), rt = sigma(4 * g + (i16 >> 2));
  const uint32_t qk_at = (uint32_t)(ra * LROW + ((g ^ (ra & 15)) << 4));
  const uint32_t qr_at = (uint32_t)(ROPE_AT + ra * 2 * R + ((g ^ ((ra >> 1) & 7)) << 4));
  const uint32_t tr_at = (uint32_t)(rt * LROW + ((((i16 & 3) >> 1) ^ (rt & 15)) << 4) + (i16 & 1) * 8);

  f32x4 o[VTILES];
#pragma unroll
  for (int t = 0; t < VTILES; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -1e30f;  // finite: a chunk that hides all its keys gives p = 0, never NaN
  float l_run = 0.f;

#pragma unroll
  for (int c = 0; c < NS - 1; ++c)
    if (begin + c < chunks) {
      look_up(begin + c);
      fetch(begin + c);
    }

  for (int c = begin; c < chunks; ++c) {
    const bool more = c + NS - 1 < chunks;
    if (more) look_up(c + NS - 1);
    // Chunk c has landed once at most the loads of the NS - 2 younger chunks are
    // in flight; where one of those has fewer loads, or is missing, all must have.
    if (partial == 0 && c + NS - 2 < chunks)
      wait_vmcnt<(NS - 2) * LOADS>();
    else
      wait_vmcnt<0>();
    block_barrier();  // every wave's part of chunk c is there, and chunk c - 1 is read
    const int loaded = min(c + NS - 1, chunks);  // chunks fetched so far
    const uint32_t bits = (good >> (KT * (loaded - 1 - c))) & ((1u << KT) - 1u);
    if (more) fetch(c + NS - 1);
    if (idle) continue;
    const uint32_t slot = ring_base + (uint32_t)((c - begin) % NS) * SLOT;

    f32x4 s[KT];
    {
      constexpr int FRAGS = KT * (KSTEPS + RSTEPS), LOOK = L == 512 ? 4 : 6;
      const uint32_t base = opaque(slot + qk_at), rope = opaque(slot + qr_at);
      x8 kf[FRAGS];
      auto load = [&](int f) {  // (step j, key tile t)
        const int j = f / KT, t = f % KT;
        kf[f] = j < KSTEPS ? *(const AFA_LDS x8*)(lds_at<uint8_t>(base ^ (uint32_t)((j & 3) << 6)) + (j >> 2) * 256 + t * 16 * LROW)
                           : *(const AFA_LDS x8*)(lds_at<uint8_t>(rope ^ (uint32_t)((j - KSTEPS) << 6)) + t * 16 * 2 * R);
      };
#pragma unroll
      for (int t = 0; t < KT; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < LOOK; ++f) load(f);
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        if (f + LOOK < FRAGS) load(f + LOOK);
        s[f % KT] = B16<DT>::mfma(kf[f], qf[f / KT], s[f % KT]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int key0 = c * KEYS;
    if (key0 + KEYS > clean_end || bits != (1u << KT) - 1u) {  // uniform
      int token, head;
      const int lim = my_row(token, head) ? visible(token) - key0 : 0;  // this row sees the chunk's keys below it
      const int quad = 4 * (int)((opaque((uint32_t)tid) >> 4) & 3u);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][i] = 16 * t + sigma(quad + i) < lim && ((bits >> t) & 1u) ? s[t][i] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
    const float m_new = fmaxf(m_run, max_over_lane_groups(top) * scale_log2);
    if (__ballot(m_new > m_run + lat_tau<DT>()) != 0ull) {
      const float alpha = fast_exp2(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int t = 0; t < VTILES; ++t) o[t] *= alpha;
      m_run = m_new;
    }
    x8 pf[KT / 2];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = fast_exp2(__builtin_fmaf(s[t][i], scale_log2, -m_run));
        l_run += p;
        pf[t / 2][4 * (t % 2) + i] = (scalar)p;
      }
    {
      constexpr int FRAGS = KT / 2 * VTILES, LOOK = 3;
      const uint32_t base = opaque(slot + tr_at);
      x4 lo[FRAGS], hi[FRAGS];
      auto load = [&](int f) {  // (32 rows ks, column tile t)
        const int ks = f / VTILES, t = f % VTILES;
        const AFA_LDS uint8_t* p = lds_at<uint8_t>(base ^ (uint32_t)((t & 7) << 5)) + (t >> 3) * 256 + ks * 32 * LROW;
        lo[f] = B16<DT>::read_tr((const AFA_LDS void*)p);
        hi[f] = B16<DT>::read_tr((const AFA_LDS void*)(p + 16 * LROW));
      };
#pragma unroll
      for (int f = 0; f < LOOK; ++f) load(f);
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        if (f + LOOK < FRAGS) load(f + LOOK);
        const x8 vf = {lo[f][0], lo[f][1], lo[f][2], lo[f][3], hi[f][0], hi[f][1], hi[f][2], hi[f][3]};
        o[f % VTILES] = B16<DT>::mfma(vf, pf[f / VTILES], o[f % VTILES]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  const float total = sum_over_lane_groups(l_run);
  int token, head;
  const bool valid = my_row(token, head);
  if (SPLIT && !whole) {
    // As the registers hold it, [16-row group][column tile][lane] of four columns: whole kilobytes per store.
    const int64_t group = (2 * (int64_t)worker + (offset == 0 ? 1 : 0)) * NW + wave;
    float* po = a.partial_o + (group * VTILES * 64 + lane) * 4;
    if (!idle) {
#pragma unroll
      for (int t = 0; t < VTILES; ++t) *(f32x4*)(po + t * 256) = o[t];
    }
    if (!idle && g == 0) *(float2*)(a.partial_ml + (group * 16 + i16) * 2) = make_float2(m_run, total);
  } else if (valid) {
    const float inv = total > 0.f ? 1.0f / total : 0.f;
    scalar* out = (scalar*)a.out + (int64_t)(start + token) * a.o_t + (int64_t)head * a.o_h + 4 * g;
#pragma unroll
    for (int t = 0; t < VTILES; ++t) {
      x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[t][i] * inv);
      *(x4*)(out + 16 * t) = v;
    }
    if (a.lse && g == 0)
      a.lse[(int64_t)(start + token) * H + head] = row_lse(m_run, total);
  }
  if (!SPLIT || left == 0) return;
  offset = 0;
  ++place;
  }
}

// Combines the parts of the tiles that several workgroups of the split form
// share: out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p, in a fixed order. A
// wave takes 16 rows and 16 * TILES columns in the layout that a wave of the main
// kernel holds them in: its lane groups first go over a quarter of the parts'
// maxima each, then every lane sums its columns over the parts, AHEAD parts of
// loads in flight. Many tiles (WAVES = 1): four such waves a workgroup, bound by
// the parts' bytes (4 L per row and part, written just before). Few tiles, whose
// parts are many: 16 waves share the parts of 16 columns and are joined through
// LDS; bound by a few dependent loads.
template <int DT, int L, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void latent_merge_kernel(LatentArgs a, int tile_rows) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x4 x4;
  constexpr int VTILES = L / 16, TILES = WAVES == 1 ? 4 : 1, AHEAD = WAVES == 1 ? 4 : 8, SHARES = VTILES / TILES;
  __shared__ f32x4 joined_o[WAVES == 1 ? 1 : WAVES][64];
  __shared__ float2 joined_sums[WAVES == 1 ? 1 : WAVES][16];
  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, i16 = lane & 15;
  const uint32_t job = WAVES == 1 ? blockIdx.x * 4u + (uint32_t)wave : blockIdx.x, groups = (uint32_t)tile_rows / 16;
  const uint32_t tile = job / (groups * SHARES), rest = job % (groups * SHARES);
  const int group = (int)(rest / SHARES), t0 = (int)(rest % SHARES) * TILES;
  if (tile >= *constant((const int32_t*)a.tile_count)) return;
  const LatentRecord record = a.records[tile];
  if (record.first == record.last || group * 16 >= record.rows) return;
  const int parts = record.last - record.first + 1, sub = WAVES == 1 ? 0 : wave;
  const int mine = (parts - sub + WAVES - 1) / WAVES;  // parts sub, sub + WAVES, ...
  auto slot = [&](int k) {
    const int p = sub + k * WAVES;
    return (2 * (int64_t)(record.first + p) + (p == 0 ? 1 : 0)) * groups + group;
  };
  auto sums = [&](int k) { return *(const float2*)(a.partial_ml + (slot(k) * 16 + i16) * 2); };

  float top = -1e30f;
#pragma unroll 4
  for (int k = g; k < mine; k += 4) top = fmaxf(top, sums(k).x);
  top = max_over_lane_groups(top);
  float total = 0.f;
  f32x4 o[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < mine; k += AHEAD) {
    float2 ml[AHEAD];
    f32x4 v[AHEAD][TILES];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int q = min(k + i, mine - 1);
      ml[i] = sums(q);
      const float* po = a.partial_o + ((slot(q) * VTILES + t0) * 64 + lane) * 4;
#pragma unroll
      for (int t = 0; t < TILES; ++t) v[i][t] = *(const f32x4*)(po + t * 256);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float weight = k + i < mine ? fast_exp2(ml[i].x - top) : 0.f;
      total += weight * ml[i].y;
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t] += weight * v[i][t];
    }
  }
  if constexpr (WAVES > 1) {
    joined_o[wave][lane] = o[0];
    if (g == 0) joined_sums[wave][i16] = make_float2(top, total);
    __syncthreads();
    if (wave != 0) return;
    const float own = top;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, joined_sums[w][i16].x);
    const float scale = fast_exp2(own - top);
    total *= scale;
    o[0] *= scale;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float2 ml = joined_sums[w][i16];
      const float weight = fast_exp2(ml.x - top);
      total += weight * ml.y;
      o[0] += weight * joined_o[w][lane];
    }
  }
  const int r = group * 16 + i16;
  if (r >= record.rows) return;
  const int packed = record.row + r, token = packed / a.H, head = packed - token * a.H;
  const float inv = total > 0.f ? 1.0f / total : 0.f;
  scalar* out = (scalar*)a.out + (int64_t)(record.start + token) * a.o_t + (int64_t)head * a.o_h + 16 * t0 + 4 * g;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[t][i] * inv);
    *(x4*)(out + 16 * t) = v;
  }
  if (a.lse && t0 == 0 && g == 0)
    a.lse[(int64_t)(record.start + token) * a.H + head] = row_lse(top, total);
}

// Expanded form (latent_attention_expanded), for prompts: keys [k_nope | k_rope]
// of 128 + 64 columns, k_nope and the values of each head, k_rope of all heads,
//   s = scale (q_nope . k_nope[h] + q_rope . k_rope),  o = softmax(s) v[h].
// 2 (128 + 64 + 128) flops a pair instead of the absorbed 2 (2 L + 64), for keys
// and values that the caller expands once per prompt. The two parts of a key are
// read from where they lie, so no concatenated, per-head copy of k_rope is made.
// One workgroup of NW waves per (request, head, NW * QT * 16 query rows), QT
// 16-row tiles a wave with Q resident; 64-key chunks of k_nope, k_rope and v
// stream through an LDS ring: three slots each, two chunks ahead, for NW = 8; two
// for NW = 4, keys two chunks ahead and values one, so that two workgroups fit a
// CU (128- or 64-row tiles: less of short, ragged or few prompts is padding or an
// idle CU, more loads per row). QK of chunk c + 1 is issued ahead of the softmax of
// chunk c, whose exponentials run in the shadow of the matrix instructions of QK
// (c + 1) and PV (c). Where even small tiles leave CUs idle, `splits` workgroups
// share a tile's keys and expanded_merge_kernel joins their float32 parts in order.
struct ExpandedArgs {
  const void* q;
  const void* k;
  const void* k_rope;
  const void* v;
  const int32_t* cu_q;
  const int32_t* cu_k;
  void* out;
  float* lse;  // [Tq][H] or NULL
  int64_t q_t, q_h, k_t, k_h, kr_t, v_t, v_h, o_t, o_h;
  int32_t Tq, Tk, B, H, causal;
  int32_t splits;
  float scale;
  float* partial_o;   // [splits][Tq * H][128], not normalised
  float* partial_ml;  // [splits][Tq * H][2]: running maximum (log2), sum of weights
};

template <int DT, int NW, int QT, bool SPLIT>
__global__ __launch_bounds__(NW * 64, NW == 8 ? 1 : 2) void expanded_kernel(ExpandedArgs a) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x8 x8;
  typedef typename B16<DT>::x4 x4;
  constexpr int BQ = NW * QT * 16, KC = 64, KT = KC / 16, NS = NW == 8 ? 3 : 2;
  constexpr int D = 128, R = 64, ROW_BYTES = 2 * D, ROPE_BYTES = 2 * R;
  constexpr int ROPE_AT = KC * ROW_BYTES, K_TILE = ROPE_AT + KC * ROPE_BYTES, V_TILE = KC * ROW_BYTES;
  constexpr int KSTEPS = D / 32, STEPS = KSTEPS + R / 32;
  // Wave loads per chunk: k_nope and v (4 rows each), k_rope (8 rows).
  constexpr int LOADS = KC / 4 / NW, ROPE_LOADS = KC / 8 / NW;
  // The whole 160 KiB for two workgroups of NW = 4: find_tile's few words lie in it too.
  __shared__ __attribute__((aligned(256))) uint8_t ring[NS * (K_TILE + V_TILE)];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, i16 = lane & 15;
  // Heads first: consecutive workgroups go to different XCDs, and a head's tiles
  // to the same one where H is a multiple of 8, which then shares its L2.
  const int head = (int)(blockIdx.x % (uint32_t)a.H);
  uint32_t index = blockIdx.x / (uint32_t)a.H;
  const int split = SPLIT ? (int)(index % (uint32_t)a.splits) : 0;
  if (SPLIT) index /= (uint32_t)a.splits;
  int request;
  uint32_t tile, tiles;
  if (!find_tile<NW * 64>(constant(a.cu_q), a.B, a.Tq, index,
                          [&](int n) { return ((uint32_t)n + BQ - 1) / BQ; }, request, tile, tiles, (uint32_t*)ring))
    return;
  __syncthreads();             // the words are read before loads land on them
  if (a.causal) tile = tiles - 1 - tile;  // the longest first
  int q_start, nq, k_start, nk;
  request_tokens(constant(a.cu_q), request, a.Tq, q_start, nq);
  request_tokens(constant(a.cu_k), request, a.Tk, k_start, nk);
  const int q0 = (int)tile * BQ;

  const scalar* Q = (const scalar*)a.q + (int64_t)q_start * a.q_t + (int64_t)head * a.q_h;
  const char* K = (const char*)a.k + 2 * ((int64_t)k_start * a.k_t + (int64_t)head * a.k_h);
  const char* KR = (const char*)a.k_rope + 2 * (int64_t)k_start * a.kr_t;
  const char* V = (const char*)a.v + 2 * ((int64_t)k_start * a.v_t + (int64_t)head * a.v_h);

  // Query i sees keys [0, nk - nq + i + 1) (causal, aligned at the end) or all.
  auto visible = [&](int i) { return a.causal ? min(max(nk - nq + i + 1, 0), nk) : nk; };
  const int kv_end = visible(min(q0 + BQ, nq) - 1);
  const int clean_end = visible(q0);
  const int all_chunks = (kv_end + KC - 1) / KC, clean_chunks = clean_end / KC;
  const int begin = SPLIT ? (int)((int64_t)all_chunks * split / a.splits) : 0;
  const int chunks = SPLIT ? (int)((int64_t)all_chunks * (split + 1) / a.splits) : all_chunks;

  x8 qf[QT][STEPS];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int row = q0 + (wave * QT + qt) * 16 + i16;
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
      qf[qt][j] = row < nq ? *(const x8*)(Q + row * a.q_t + 32 * j + 8 * g) : __builtin_bit_cast(x8, u32x4{0u, 0u, 0u, 0u});
  }

  const uint32_t ring_base = lds_address(ring);
  auto k_slot = [&](int chunk) { return opaque_uniform(ring_base + (uint32_t)(chunk % NS) * K_TILE); };
  auto v_slot = [&](int chunk) { return opaque_uniform(ring_base + (uint32_t)(NS * K_TILE) + (uint32_t)(chunk % NS) * V_TILE); };
  auto load = [](uint32_t to, uint32_t off, const char* from) {
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(off), "s"(from) : "memory");
  };
  // Rows of 128 columns: load p of this wave lands on rows 4 (wave * LOADS + p) ..
  // + 3, unit u of row r at u ^ (r & 15). Rows past the last key read the last key instead
  // (masked later). 32-bit row offsets: the host holds 64 rows below 2^31 bytes.
  const uint32_t k_row = (uint32_t)(2 * a.k_t), v_row = (uint32_t)(2 * a.v_t), r_row = (uint32_t)(2 * a.kr_t);
  auto fetch_rows = [&](uint32_t slot, const char* rows, uint32_t row_bytes, int key0) {
    const char* base = rows + (int64_t)key0 * row_bytes;
    const int last = nk - 1 - key0;
    const uint32_t ln = opaque((uint32_t)tid) & 63u;
#pragma unroll
    for (int p = 0; p < LOADS; ++p) {
      const int r = (wave * LOADS + p) * 4 + (int)(ln >> 4);
      load(slot + (uint32_t)((wave * LOADS + p) * 4 * ROW_BYTES),
           (uint32_t)min(r, last) * row_bytes + (((ln & 15u) ^ (uint32_t)(r & 15)) << 4), base);
    }
  };
  auto fetch_k = [&](int chunk) {
    const int key0 = chunk * KC;
    const uint32_t slot = k_slot(chunk);
    fetch_rows(slot, K, k_row, key0);
    const char* base = KR + (int64_t)key0 * r_row;
    const int last = nk - 1 - key0;
    const uint32_t ln = opaque((uint32_t)tid) & 63u;
#pragma unroll
    for (int p = 0; p < ROPE_LOADS; ++p) {
      const int r = (wave * ROPE_LOADS + p) * 8 + (int)(ln >> 3);
      load(slot + (uint32_t)(ROPE_AT + (wave * ROPE_LOADS + p) * 8 * ROPE_BYTES),
           (uint32_t)min(r, last) * r_row + (((ln & 7u) ^ (uint32_t)((r >> 1) & 7)) << 4), base);
    }
  };
  auto fetch_v = [&](int chunk) { fetch_rows(v_slot(chunk), V, v_row, chunk * KC); };

  const int ra = sigma(i16), rt = sigma(4 * g + (i16 >> 2));
  const uint32_t qk_at = (uint32_t)(ra * ROW_BYTES + ((g ^ (ra & 15)) << 4));
  const uint32_t qr_at = (uint32_t)(ROPE_AT + ra * ROPE_BYTES + ((g ^ ((ra >> 1) & 7)) << 4));
  const uint32_t tr_at = (uint32_t)(rt * ROW_BYTES + ((((i16 & 3) >> 1) ^ (rt & 15)) << 4) + (i16 & 1) * 8);

  f32x4 o[QT][D / 16];
  float m_run[QT], l_run[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m_run[qt] = -1e30f;
    l_run[qt] = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale_log2 = a.scale * LAT_LOG2E;

  constexpr int QK_FRAGS = STEPS * KT, LOOK = 5;
  auto qk_chunk = [&](int chunk, f32x4 (&s)[KT][QT], auto&& between) {
    const uint32_t slot = k_slot(chunk);
    const uint32_t base = opaque(slot + qk_at), rope = opaque(slot + qr_at);
    x8 kf[QK_FRAGS];
    auto load = [&](int f) {  // (step j, key tile t)
      const int j = f / KT, t = f % KT;
      kf[f] = j < KSTEPS ? *(const AFA_LDS x8*)(lds_at<uint8_t>(base ^ (uint32_t)(j << 6)) + t * 16 * ROW_BYTES)
                         : *(const AFA_LDS x8*)(lds_at<uint8_t>(rope ^ (uint32_t)((j - KSTEPS) << 6)) + t * 16 * ROPE_BYTES);
    };
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[t][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < LOOK; ++f) load(f);
#pragma unroll
    for (int f = 0; f < QK_FRAGS; ++f) {
      if (f + LOOK < QK_FRAGS) load(f + LOOK);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[f % KT][qt] = B16<DT>::mfma(kf[f], qf[qt][f / KT], s[f % KT][qt]);
      between(f);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int PV_FRAGS = (KC / 32) * (D / 16);
  auto pv_chunk = [&](int chunk, x8 (&pf)[QT][KC / 32], auto&& between) {
    const uint32_t base = opaque(v_slot(chunk) + tr_at);
    constexpr int VLOOK = 3;
    x4 lo[PV_FRAGS], hi[PV_FRAGS];
    auto load = [&](int f) {  // (32 keys ks, column tile t)
      const int ks = f / (D / 16), t = f % (D / 16);
      const AFA_LDS uint8_t* p = lds_at<uint8_t>(base ^ (uint32_t)(t << 5)) + ks * 32 * ROW_BYTES;
      lo[f] = B16<DT>::read_tr((const AFA_LDS void*)p);
      hi[f] = B16<DT>::read_tr((const AFA_LDS void*)(p + 16 * ROW_BYTES));
    };
#pragma unroll
    for (int f = 0; f < VLOOK; ++f) load(f);
#pragma unroll
    for (int f = 0; f < PV_FRAGS; ++f) {
      if (f + VLOOK < PV_FRAGS) load(f + VLOOK);
      const int ks = f / (D / 16), t = f % (D / 16);
      const x8 vf = {lo[f][0], lo[f][1], lo[f][2], lo[f][3], hi[f][0], hi[f][1], hi[f][2], hi[f][3]};
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) o[qt][t] = B16<DT>::mfma(vf, pf[qt][ks], o[qt][t]);
      between(f);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto mask = [&](int chunk, f32x4 (&s)[KT][QT]) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int row = q0 + (wave * QT + qt) * 16 + (int)(opaque((uint32_t)tid) & 15u);
      const int lim = visible(min(row, nq - 1)) - chunk * KC;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][qt][i] = 16 * t + sigma(4 * g + i) < lim ? s[t][qt][i] : -INFINITY;
    }
  };

  constexpr int HALF = QT * 8, QK_EXP0 = QT + 2, PV_EXP_STEPS = PV_FRAGS / 2 - 1;
  f32x4 s_a[KT][QT], s_b[KT][QT];
  if (begin < chunks) {
    fetch_k(begin);
    fetch_v(begin);
    if (begin + 1 < chunks) {
      fetch_k(begin + 1);
      if constexpr (NS == 3) fetch_v(begin + 1);
      wait_vmcnt<LOADS + ROPE_LOADS + (NS == 3 ? LOADS : 0)>();
    } else {
      wait_vmcnt<0>();
    }
    block_barrier();
    qk_chunk(begin, s_a, [](int) {});
  }
  auto iteration = [&](int c, f32x4 (&cur)[KT][QT], f32x4 (&nxt)[KT][QT]) {
    // Keys of chunk c + 1 and values of c have landed, and every wave is past QK (c)
    // and PV (c - 1), whose slots are free.
    wait_vmcnt<0>();
    block_barrier();
    if (c + 2 < chunks) fetch_k(c + 2);
    if (c + NS - 1 < chunks) fetch_v(c + NS - 1);
    if (c >= clean_chunks) mask(c, cur);
    x8 pf[QT][KC / 32];
    float top[QT], m_new[QT], psum[QT];
    auto exp_element = [&](int e) {  // (half, qt, key tile of the half, i)
      const int h = e / HALF, qt = (e / 8) % QT, t = 2 * h + (e / 4) % 2, i = e % 4;
      const float p = fast_exp2(__builtin_fmaf(cur[t][qt][i], scale_log2, -m_run[qt]));
      psum[qt] += p;
      pf[qt][h][(t & 1) * 4 + i] = (scalar)p;
    };
    auto qk_between = [&](int f) {
      if (f == QK_FRAGS / 2 - 1) __builtin_amdgcn_s_setprio(2);
      if (f < QT) {
        float m = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) m = fmaxf(m, cur[t][f][i]);
        top[f] = m;
      } else if (f == QT) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          m_new[qt] = fmaxf(m_run[qt], max_over_lane_groups(top[qt]) * scale_log2);
          psum[qt] = 0.f;
        }
      } else if (f == QT + 1) {
        bool grow = false;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) grow |= m_new[qt] > m_run[qt] + lat_tau<DT>();
        if (__ballot(grow) != 0ull) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            const float alpha = fast_exp2(m_run[qt] - m_new[qt]);
            l_run[qt] *= alpha;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) o[qt][t] *= alpha;
            m_run[qt] = m_new[qt];
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < HALF; ++e)
          if (QK_EXP0 + e * (QK_FRAGS - QK_EXP0) / HALF == f) exp_element(e);
      }
    };
    auto pv_between = [&](int f) {
      if (f == PV_FRAGS / 2 - 1) __builtin_amdgcn_s_setprio(0);
      if (f < PV_EXP_STEPS) {
#pragma unroll
        for (int e = 0; e < HALF; ++e)
          if (e * PV_EXP_STEPS / HALF == f) exp_element(HALF + e);
      } else if (f == PV_EXP_STEPS + 1) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) l_run[qt] += psum[qt];
      }
    };
    // Wave priority steps down with the wave's progress through a chunk: of the
    // two waves of a SIMD the one behind wins. The last chunk also runs a QK,
    // over a slot that no load is in flight into; nobody reads those scores.
    __builtin_amdgcn_s_setprio(3);
    qk_chunk(c + 1, nxt, qk_between);
    __builtin_amdgcn_s_setprio(1);
    pv_chunk(c, pf, pv_between);
  };
  for (int c = begin; c < chunks; c += 2) {
    iteration(c, s_a, s_b);
    if (c + 1 < chunks) iteration(c + 1, s_b, s_a);
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int row = q0 + (wave * QT + qt) * 16 + i16;
    const float total = sum_over_lane_groups(l_run[qt]);
    if (row >= nq) continue;
    if constexpr (SPLIT) {
      const int64_t at = ((int64_t)split * a.Tq + q_start + row) * a.H + head;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) *(f32x4*)(a.partial_o + at * D + 16 * t + 4 * g) = o[qt][t];
      if (g == 0) *(float2*)(a.partial_ml + at * 2) = make_float2(m_run[qt], total);
    } else {
      const float inv = total > 0.f ? 1.0f / total : 0.f;
      scalar* out = (scalar*)a.out + (int64_t)(q_start + row) * a.o_t + (int64_t)head * a.o_h + 4 * g;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[qt][t][i] * inv);
        *(x4*)(out + 16 * t) = v;
      }
      if (a.lse && g == 0)
        a.lse[(int64_t)(q_start + row) * a.H + head] = row_lse(m_run[qt], total);
    }
  }
}

// Joins the parts of split keys, in order: half a wave per (query, head) row, four
// columns a lane, four parts of loads in flight.
template <int DT>
__global__ __launch_bounds__(256) void expanded_merge_kernel(ExpandedArgs a) {
  typedef typename B16<DT>::scalar scalar;
  typedef typename B16<DT>::x4 x4;
  constexpr int AHEAD = 4;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (int64_t)a.Tq * a.H;
  const int column = 4 * (threadIdx.x & 31);
  const int end = min(max(constant(a.cu_q)[a.B], 0), a.Tq);  // rows of no request stay as they are
  if (row >= rows || row / a.H >= end || row / a.H < constant(a.cu_q)[0]) return;
  float top = -1e30f;
  for (int p = 0; p < a.splits; ++p) top = fmaxf(top, a.partial_ml[(p * rows + row) * 2]);
  float total = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < a.splits; p += AHEAD) {
    float2 ml[AHEAD];
    f32x4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int64_t at = min(p + i, a.splits - 1) * rows + row;
      ml[i] = *(const float2*)(a.partial_ml + at * 2);
      v[i] = *(const f32x4*)(a.partial_o + at * 128 + column);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float weight = p + i < a.splits ? fast_exp2(ml[i].x - top) : 0.f;
      total += weight * ml[i].y;
      o += weight * v[i];
    }
  }
  const float inv = total > 0.f ? 1.0f / total : 0.f;
  x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (scalar)(o[i] * inv);
  *(x4*)((scalar*)a.out + row / a.H * a.o_t + row % a.H * a.o_h + column) = v;
  if (a.lse && column == 0) a.lse[row] = row_lse(top, total);
}

namespace {

// Whether a launch, which counts its threads in 32 bits, can have so many workgroups.
bool launchable(int64_t workgroups, int threads) { return workgroups <= 0xffffffffll / threads; }

bool rows_fit(const void* p, int64_t a, int64_t b) { return ((uintptr_t)p & 15) == 0 && (a | b) % 8 == 0; }

int check_latent(const LatentParams* p) {
  if (!p) return AFA_E_NULL;
  if (p->dtype != AFA_DTYPE_BF16 && p->dtype != AFA_DTYPE_F16) return AFA_E_DTYPE;
  if (p->T < 0 || p->B <= 0 || p->H <= 0 || p->W <= 0 || p->BLOCKS <= 0) return AFA_E_SHAPE;
  if ((p->L != 128 && p->L != 256 && p->L != 512) || (p->R != 0 && p->R != 64)) return AFA_E_SHAPE;
  if (p->PAGE < 16 || p->PAGE > (1 << 20) || (p->PAGE & (p->PAGE - 1))) return AFA_E_SHAPE;
  // Packed rows, tiles and positions are 32-bit numbers.
  if ((int64_t)p->T * p->H > 0x7fffff00ll || (int64_t)p->W * p->PAGE > 0x7fffff00ll || p->B > 0x3fffffff) return AFA_E_SHAPE;
  if (!(p->scale > 0.0f) || !std::isfinite(p->scale)) return AFA_E_SHAPE;
  return AFA_OK;
}

constexpr int LAT_CUS = 256;
constexpr int64_t LAT_STREAM_BYTES = 128ll << 20;
// Merge jobs of 16 waves each up to here, of one wave above: one request of 4K rows
// (256 jobs) 23.5 and 27.7 us, of 64K rows 45 and 144; 16 of 4K rows with 16 heads (2560)
// 31.8 and 30.5, 8 x 4 tokens of 64 heads over 4K rows (6144) 78 and 47.
constexpr int64_t LAT_FEW_JOBS = 2048;

// Form of a call: waves (of 16 rows each) of a tile, 8 where a request has more
// than 64 rows on average, else 4 (64 decode requests of 8000 rows, 128 heads 170 us
// with 8, 195 with 4; 4 chunks of 512 behind 8K 4079 and 4403; one of 4096 rows
// 30.5 and 30.8); and workgroups of the split form, one per CU or two, 0 for the
// form of one tile per workgroup: where the tiles (at most rows / tile + B of
// them) would fill the GPU four times over anyway, or a single request's fill 85%
// of their rounds (128 heads behind 8000 rows: 230 tokens 460 us directly, 461
// split; 500 tokens 971 and 989; 400 tokens, whose second round is half empty, 890
// and 856; 1000 tokens with no context 180 and 186).
struct LatentPlan {
  int waves;
  int workers;
  int64_t tiles;
  bool stream;  // split form: a tile or less per request on average, a cache of 128 MiB or more
};
LatentPlan plan_latent(const LatentParams* p) {
  LatentPlan plan;
  plan.waves = ((int64_t)p->T + p->B - 1) / p->B * p->H > 64 ? 8 : 4;
  plan.tiles = (int64_t)p->T * p->H / (16 * plan.waves) + p->B;
  const int slots = plan.waves == 8 ? LAT_CUS : 2 * LAT_CUS;
  const int64_t single = ((int64_t)p->T * p->H + 16 * plan.waves - 1) / (16 * plan.waves);  // a single request's tiles
  const bool even = p->B == 1 && 20 * single >= 17 * ((single + slots - 1) / slots) * slots;
  plan.workers = plan.tiles <= 4 * slots && !even ? slots : 0;
  plan.stream = (int64_t)p->T * p->H <= (int64_t)p->B * 16 * plan.waves &&
                (int64_t)p->BLOCKS * p->PAGE * (p->L + p->R) * 2 >= LAT_STREAM_BYTES;
  return plan;
}

// Merge jobs of 16 rows and 16 columns.
int64_t latent_merge_jobs(const LatentPlan& plan, int L) { return plan.tiles * plan.waves * (L / 16); }

// Workspace of the split form: parts, their maxima and sums, records, the count of tiles.
int64_t latent_part_rows(const LatentPlan& plan) { return 2ll * plan.workers * 16 * plan.waves; }
uint64_t latent_bytes(const LatentParams* p, const LatentPlan& plan) {
  if (plan.workers == 0 || p->T == 0) return 0;
  return (uint64_t)(latent_part_rows(plan) * (p->L + 2) * 4 + plan.tiles * (int64_t)sizeof(LatentRecord) + 16);
}

template <int DT, int L, int R>
int launch_latent(LatentArgs a, const LatentPlan& plan, void* workspace, hipStream_t s) {
  if (!launchable(plan.tiles, 64 * plan.waves)) return AFA_E_SHAPE;
  if (plan.workers == 0) {
    const dim3 grid((unsigned)plan.tiles);
    if (plan.waves == 8)
      hipLaunchKernelGGL((latent_kernel<DT, L, R, 8, false, false>), grid, dim3(512), 0, s, a);
    else
      hipLaunchKernelGGL((latent_kernel<DT, L, R, 4, false, false>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
  }
  const int64_t part_rows = latent_part_rows(plan);
  a.workers = plan.workers;
  a.partial_o = (float*)workspace;
  a.partial_ml = a.partial_o + part_rows * L;
  a.tile_count = (uint32_t*)(a.partial_ml + part_rows * 2);
  a.records = (LatentRecord*)(a.tile_count + 4);
  a.tiles = (uint32_t)plan.tiles;
  const dim3 grid((unsigned)plan.workers);
  if (plan.waves == 8 && plan.stream)
    hipLaunchKernelGGL((latent_kernel<DT, L, R, 8, true, true>), grid, dim3(512), 0, s, a);
  else if (plan.waves == 8)
    hipLaunchKernelGGL((latent_kernel<DT, L, R, 8, true, false>), grid, dim3(512), 0, s, a);
  else if (plan.stream)
    hipLaunchKernelGGL((latent_kernel<DT, L, R, 4, true, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((latent_kernel<DT, L, R, 4, true, false>), grid, dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  const int rows = 16 * plan.waves;
  const int64_t jobs = latent_merge_jobs(plan, L);
  if (jobs <= LAT_FEW_JOBS)
    hipLaunchKernelGGL((latent_merge_kernel<DT, L, 16>), dim3((unsigned)jobs), dim3(1024), 0, s, a, rows);
  else
    hipLaunchKernelGGL((latent_merge_kernel<DT, L, 1>), dim3((unsigned)((jobs / 4 + 3) / 4)), dim3(256), 0, s, a, rows);
  return (int)hipGetLastError();
}

template <int DT>
int dispatch_latent(const LatentArgs& a, const LatentParams* p, const LatentPlan& plan, void* workspace, hipStream_t s) {
  if (p->R == 64) {
    if (p->L == 512) return launch_latent<DT, 512, 64>(a, plan, workspace, s);
    if (p->L == 256) return launch_latent<DT, 256, 64>(a, plan, workspace, s);
    return launch_latent<DT, 128, 64>(a, plan, workspace, s);
  }
  if (p->L == 512) return launch_latent<DT, 512, 0>(a, plan, workspace, s);
  if (p->L == 256) return launch_latent<DT, 256, 0>(a, plan, workspace, s);
  return launch_latent<DT, 128, 0>(a, plan, workspace, s);
}

}  // namespace
}  // namespace afa

extern "C" int launch_latent_attention(void* stream, const void* q, const void* q_rope, const void* kv_cache,
                                       const int32_t* block_table, const int32_t* cu_seqlens_q, const int32_t* seqused_kv,
                                       void* out, float* softmax_lse, void* workspace, uint64_t workspace_bytes,
                                       const LatentParams* p) {
  using namespace afa;
  const int status = check_latent(p);
  if (status) return status;
  if (!q || !kv_cache || !block_table || !cu_seqlens_q || !seqused_kv || !out || (p->R && !q_rope)) return AFA_E_NULL;
  if (p->T == 0) return AFA_OK;
  if (!rows_fit(q, p->q_stride_t, p->q_stride_h) || !rows_fit(out, p->out_stride_t, p->out_stride_h) ||
      (p->R && !rows_fit(q_rope, p->q_rope_stride_t, p->q_rope_stride_h)) || !rows_fit(kv_cache, 0, 0))
    return AFA_E_SHAPE;
  const LatentPlan plan = plan_latent(p);
  const uint64_t need = latent_bytes(p, plan);
  if (need > 0 && (!workspace || workspace_bytes < need)) return AFA_E_WORKSPACE;
  if ((uintptr_t)workspace & 15) return AFA_E_WORKSPACE;
  LatentArgs a = {};
  a.q = q;
  a.q_rope = q_rope;
  a.cache = kv_cache;
  a.table = block_table;
  a.cu = cu_seqlens_q;
  a.used = seqused_kv;
  a.out = out;
  a.lse = softmax_lse;
  a.q_t = p->q_stride_t;
  a.q_h = p->q_stride_h;
  a.qr_t = p->q_rope_stride_t;
  a.qr_h = p->q_rope_stride_h;
  a.o_t = p->out_stride_t;
  a.o_h = p->out_stride_h;
  a.T = p->T;
  a.B = p->B;
  a.H = p->H;
  a.W = p->W;
  a.page_shift = __builtin_ctz((unsigned)p->PAGE);
  a.blocks = p->BLOCKS;
  a.causal = p->causal ? 1 : 0;
  a.scale = p->scale;
  return p->dtype == AFA_DTYPE_F16 ? dispatch_latent<DT_F16>(a, p, plan, workspace, (hipStream_t)stream)
                                   : dispatch_latent<DT_BF16>(a, p, plan, workspace, (hipStream_t)stream);
}

extern "C" int workspace_size_latent_attention(uint64_t* bytes, const LatentParams* p) {
  using namespace afa;
  if (!bytes) return AFA_E_NULL;
  const int status = check_latent(p);
  if (status) return status;
  *bytes = latent_bytes(p, plan_latent(p));
  return AFA_OK;
}

extern "C" int form_latent_attention(int64_t form[2], const LatentParams* p) {
  using namespace afa;
  if (!form) return AFA_E_NULL;
  const int status = check_latent(p);
  if (status) return status;
  const LatentPlan plan = plan_latent(p);
  form[0] = 16 * plan.waves;
  form[1] = plan.workers;
  return AFA_OK;
}

extern "C" int split_form_latent_attention(int64_t form[2], const LatentParams* p) {
  using namespace afa;
  if (!form) return AFA_E_NULL;
  const int status = check_latent(p);
  if (status) return status;
  const LatentPlan plan = plan_latent(p);
  form[0] = plan.workers > 0 && plan.stream ? 1 : 0;
  form[1] = plan.workers == 0 ? 0 : latent_merge_jobs(plan, p->L) <= LAT_FEW_JOBS ? 16 : 1;
  return AFA_OK;
}

namespace afa {
namespace {

// Form of an expanded call: rows of a tile (256, 128 or 64) and key splits.
struct ExpandedPlan {
  int rows;
  int splits;
};

int check_expanded(const LatentExpandedParams* p) {
  if (!p) return AFA_E_NULL;
  if (p->dtype != AFA_DTYPE_BF16 && p->dtype != AFA_DTYPE_F16) return AFA_E_DTYPE;
  if (p->Tq < 0 || p->Tk < 0 || p->B <= 0 || p->H <= 0 || p->Tq > 0x7fffff00 || p->Tk > 0x7fffff00) return AFA_E_SHAPE;
  if (p->D != 128 || p->R != 64 || !(p->scale > 0.0f) || !std::isfinite(p->scale)) return AFA_E_SHAPE;
  if (((int64_t)p->Tq / 64 + p->B) * p->H > 0x7fffffffll / EXP_MAX_SPLITS) return AFA_E_SHAPE;
  return AFA_OK;
}

// The form that a cost model finds cheapest (us), fixed at 256 CUs, with mean
// request lengths (the launcher reads no device memory). A tile's 64-key chunk
// costs ALONE where it has its CU to itself and FULL with the CU's workgroups at
// work (one of 256 rows, two of 128 or 64); a round of workgroups START. Measured
// at 256 / 128 / 64 rows, bfloat16: 1 x 8192 causal, 32 heads 648 / 666 / 854 us; 1 x 1500,
// 128 heads 132 / 127 / 159; 5 x 235..470 behind up to 2000, 16 heads 74 / 56 / 47;
// 1 x 2048, 16 heads 75 / 56 / 46. Split keys add a launch and their float32 parts
// written and read at 3 TB/s: 64 rows in 1 / 2 / 4 / 8 parts, 8 x 20 behind 3000, 8 heads
// 55 / 35 / 26 / 28; 1 x 500 behind 4000, 32 heads 82 / 67 / 79 / 101; one query of 8192
// keys, 16 heads 133 / 77 / 42 / 26.5 (22.5 in 16).
ExpandedPlan plan_expanded(const LatentExpandedParams* p) {
  constexpr int FORMS = 3, ROWS[FORMS] = {256, 128, 64}, SLOTS[FORMS] = {256, 512, 512};
  constexpr double ALONE[FORMS] = {2.0, 1.5, 1.2}, FULL[FORMS] = {2.85, 2.9, 1.65}, START[FORMS] = {12.0, 11.0, 7.5};
  constexpr double MERGE = 5.0, MERGE_RATE = 3e6;  // us, bytes a us
  const int64_t nq = std::max<int64_t>(1, (p->Tq + p->B - 1) / p->B), nk = std::max<int64_t>(1, (p->Tk + p->B - 1) / p->B);
  const double chunks = std::ceil(nk / 64.0);
  // Mean keys of a query over those of the last.
  const double mean = p->causal && nk > 1 ? 1.0 - 0.5 * std::min(1.0, (double)(nq - 1) / nk) : 1.0;
  auto cost = [&](int form, int splits) {
    const double blocks = (double)((nq + ROWS[form] - 1) / ROWS[form]) * p->B * p->H * splits;
    const double rounds = blocks / SLOTS[form], each = std::ceil(chunks / splits);
    const double full = (p->causal ? rounds : std::ceil(rounds)) * mean * each * FULL[form] *
                        std::min(1.0, std::max(rounds, 256.0 / SLOTS[form]));
    return START[form] * (0.5 + 0.5 * std::ceil(rounds)) + std::max(each * ALONE[form], full) +
           (splits > 1 ? MERGE + (double)splits * p->Tq * p->H * (2 * 130 * 4) / MERGE_RATE : 0.0);
  };
  ExpandedPlan plan{ROWS[0], 1};
  double best = cost(0, 1);
  for (int form = 1; form < FORMS; ++form)
    if (cost(form, 1) < best) {
      best = cost(form, 1);
      plan.rows = ROWS[form];
    }
  const int64_t most = std::min<int64_t>(EXP_MAX_SPLITS, (int64_t)chunks / 4);  // at least 256 keys each
  for (int splits = 2; splits <= most; ++splits)
    if (cost(2, splits) < best) {
      best = cost(2, splits);
      plan = ExpandedPlan{64, splits};
    }
  return plan;
}

uint64_t expanded_bytes(const LatentExpandedParams* p, const ExpandedPlan& plan) {
  return plan.splits > 1 ? (uint64_t)plan.splits * p->Tq * p->H * (128 + 2) * 4 : 0;
}

template <int DT>
int launch_expanded(const ExpandedArgs& a, const ExpandedPlan& plan, hipStream_t s) {
  const int64_t workgroups = ((int64_t)a.Tq / plan.rows + a.B) * a.H * plan.splits;
  const int64_t merge = ((int64_t)a.Tq * a.H + 7) / 8;
  if (!launchable(workgroups, plan.rows == 256 ? 512 : 256) || (plan.splits > 1 && !launchable(merge, 256))) return AFA_E_SHAPE;
  const dim3 grid((unsigned)workgroups);
  if (plan.splits > 1)
    hipLaunchKernelGGL((expanded_kernel<DT, 4, 1, true>), grid, dim3(256), 0, s, a);
  else if (plan.rows == 256)
    hipLaunchKernelGGL((expanded_kernel<DT, 8, 2, false>), grid, dim3(512), 0, s, a);
  else if (plan.rows == 128)
    hipLaunchKernelGGL((expanded_kernel<DT, 4, 2, false>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((expanded_kernel<DT, 4, 1, false>), grid, dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.splits == 1) return (int)e;
  hipLaunchKernelGGL(expanded_merge_kernel<DT>, dim3((unsigned)merge), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace afa

extern "C" int launch_latent_attention_expanded(void* stream, const void* q, const void* k_nope, const void* k_rope,
                                                const void* v, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                                void* out, float* softmax_lse, void* workspace, uint64_t workspace_bytes,
                                                const LatentExpandedParams* p) {
  using namespace afa;
  const int status = check_expanded(p);
  if (status) return status;
  if (!q || !cu_seqlens_q || !cu_seqlens_k || !out || (p->Tk > 0 && (!k_nope || !k_rope || !v))) return AFA_E_NULL;
  if (!rows_fit(q, p->q_stride_t, p->q_stride_h) || !rows_fit(out, p->out_stride_t, p->out_stride_h) ||
      !rows_fit(k_nope, p->k_stride_t, p->k_stride_h) || !rows_fit(k_rope, p->k_rope_stride_t, 0) ||
      !rows_fit(v, p->v_stride_t, p->v_stride_h))
    return AFA_E_SHAPE;
  for (int64_t stride : {p->k_stride_t, p->k_rope_stride_t, p->v_stride_t})
    if (stride < 0 || stride >= (1ll << 23)) return AFA_E_SHAPE;  // 64 rows span less than 2^31 bytes
  if (p->Tq == 0) return AFA_OK;
  const ExpandedPlan plan = plan_expanded(p);
  const uint64_t need = expanded_bytes(p, plan);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return AFA_E_WORKSPACE;
  ExpandedArgs a;
  a.q = q;
  a.k = k_nope;
  a.k_rope = k_rope;
  a.v = v;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.out = out;
  a.lse = softmax_lse;
  a.q_t = p->q_stride_t;
  a.q_h = p->q_stride_h;
  a.k_t = p->k_stride_t;
  a.k_h = p->k_stride_h;
  a.kr_t = p->k_rope_stride_t;
  a.v_t = p->v_stride_t;
  a.v_h = p->v_stride_h;
  a.o_t = p->out_stride_t;
  a.o_h = p->out_stride_h;
  a.Tq = p->Tq;
  a.Tk = p->Tk;
  a.B = p->B;
  a.H = p->H;
  a.causal = p->causal ? 1 : 0;
  a.splits = plan.splits;
  a.scale = p->scale;
  a.partial_o = (float*)workspace;
  a.partial_ml = (float*)workspace + (need ? (int64_t)plan.splits * p->Tq * p->H * 128 : 0);
  return p->dtype == AFA_DTYPE_F16 ? launch_expanded<DT_F16>(a, plan, (hipStream_t)stream)
                                   : launch_expanded<DT_BF16>(a, plan, (hipStream_t)stream);
}

extern "C" int workspace_size_latent_attention_expanded(uint64_t* bytes, const LatentExpandedParams* p) {
  using namespace afa;
  if (!bytes) return AFA_E_NULL;
  const int status = check_expanded(p);
  if (status) return status;
  *bytes = expanded_bytes(p, plan_expanded(p));
  return AFA_OK;
}

extern "C" int form_latent_attention_expanded(int64_t form[2], const LatentExpandedParams* p) {
  using namespace afa;
  if (!form) return AFA_E_NULL;
  const int status = check_expanded(p);
  if (status) return status;
  const ExpandedPlan plan = plan_expanded(p);
  form[0] = plan.rows;
  form[1] = plan.splits;
  return AFA_OK;
}
