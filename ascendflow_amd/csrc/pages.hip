// Upkeep of a paged cache's pages, for gfx950: copies, forks of requests (with copies
// on write, releases and reservations) and compaction.
//
// A table row [W] names the pages of one request, -1 where it has none; `counts` holds
// the number of references of each page, 0 for a free one. Everything is integers and
// comparisons: what a call gives follows from its operands alone, whatever the order of
// its atomics. Copies are bound by HBM (500 pages of 64 KiB in 16 caches 180 us, 5.1 TB/s);
// the others by launches and chains of dependent loads over a table and a list of counts
// that fit the L2s: a fork of 32 rows 3.4 and 9.8 us, of 256 rows of 1024 pages 2.9 and 15,
// a compaction of 2048 pages 5.8 and 2.1, of 300000 4.1, 8.5 and 3.2.
#include <algorithm>

#include "common.h"
#include "../../include/ascendflow_amd.h"

namespace afa {

// ---- copies --------------------------------------------------------------------

constexpr int COPY_CACHES = 64;          // of a launch
constexpr int COPY_BYTES = 256 * 16 * 4; // of a workgroup: four 16-byte pieces a thread

struct CopyArgs {
  const int32_t* source;
  const int32_t* destination;
  int32_t blocks, parts;
  uint8_t* cache[COPY_CACHES];
  uint64_t bytes[COPY_CACHES];  // of a page
};

// One workgroup per (pair, part of COPY_BYTES, cache). Pieces of 16 bytes, or of 4 or 1
// where pages do not lie on 16 or 4.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const uint32_t pair = blockIdx.x / (uint32_t)a.parts, part = blockIdx.x % (uint32_t)a.parts;
  const uint64_t bytes = a.bytes[blockIdx.y], at = (uint64_t)part * COPY_BYTES;
  if (at >= bytes) return;
  const int32_t from = a.source[pair], to = a.destination[pair];
  if (from < 0 || from >= a.blocks || to < 0 || to >= a.blocks || from == to) return;
  const uint8_t* src = a.cache[blockIdx.y] + (uint64_t)from * bytes + at;
  uint8_t* dst = a.cache[blockIdx.y] + (uint64_t)to * bytes + at;
  const uint32_t n = (uint32_t)min(bytes - at, (uint64_t)COPY_BYTES);
  const uint64_t off = (uint64_t)(uintptr_t)a.cache[blockIdx.y] | bytes;
  if (off % 16 == 0) {
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t o = (threadIdx.x + 256u * i) * 16u;
      if (o < n) v[i] = *(const u32x4*)(src + o);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t o = (threadIdx.x + 256u * i) * 16u;
      if (o < n) *(u32x4*)(dst + o) = v[i];
    }
  } else if (off % 4 == 0) {
    for (uint32_t o = threadIdx.x * 4u; o < n; o += 1024u) *(uint32_t*)(dst + o) = *(const uint32_t*)(src + o);
  } else {
    for (uint32_t o = threadIdx.x; o < n; o += 256u) dst[o] = src[o];
  }
}

// ---- tables --------------------------------------------------------------------

constexpr int TABLE_THREADS = 1024;
constexpr int FORK_MAX_B = 8192;

struct ForkArgs {
  int32_t* table;
  int32_t* counts;
  const int32_t* parents;
  const int32_t* used;
  int32_t* source;
  int32_t* destination;
  int32_t* missing;
  int32_t* rows;      // workspace [B][W]: rows of other parents
  int32_t* tails;     // workspace [B]
  int32_t* free_list; // workspace [BLOCKS]
  int32_t B, W, BLOCKS, page_shift, reserve;
};

__device__ __forceinline__ bool names_page(int32_t entry, int32_t blocks) { return (uint32_t)entry < (uint32_t)blocks; }

__device__ __forceinline__ int load_count(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sizes of row b: whether it lives, pages that its tokens take and those it wants, not held to the table.
struct ForkRow {
  int32_t parent;
  int64_t used, held, most;
  __device__ __forceinline__ ForkRow(const ForkArgs& a, int b) {
    parent = a.parents[b];
    if ((uint32_t)parent >= (uint32_t)a.B) parent = -1;
    const int64_t page = (int64_t)1 << a.page_shift;
    used = max(a.used[b], 0);
    held = (used + page - 1) >> a.page_shift;
    most = (used + a.reserve + page - 1) >> a.page_shift;
  }
};

// Each row from its parent's, into the workspace (but for what a row keeps of its own), the references that change
// with it, and the page that it will go on writing to, -1 where its next token starts a page.
__global__ __launch_bounds__(256) void fork_rows_kernel(ForkArgs a) {
  const int b = (int)blockIdx.y;
  const ForkRow row(a, b);
  const int column = (int)(blockIdx.x * 256 + threadIdx.x);
  if (column >= a.W) return;
  const int64_t at = (int64_t)b * a.W + column;
  const int32_t old = a.table[at];
  int32_t now = -1;
  if (row.parent >= 0 && column < row.held) now = row.parent == b ? old : a.table[(int64_t)row.parent * a.W + column];
  if (column == min(row.held, (int64_t)a.W) - 1 || (row.held == 0 && column == 0)) {
    const bool partial = row.parent >= 0 && (row.used & ((1 << a.page_shift) - 1)) && row.held <= a.W;
    a.tails[b] = partial && names_page(now, a.BLOCKS) ? now : -1;
  }
  if (row.parent != b) a.rows[at] = now;
  if (old == now) return;
  if (names_page(old, a.BLOCKS)) atomicSub(a.counts + old, 1);
  if (names_page(now, a.BLOCKS)) atomicAdd(a.counts + now, 1);
}

// Exclusive sum over the workgroup's threads and, in `total`, the sum of all; words: TABLE_THREADS / 64 of LDS.
__device__ __forceinline__ int block_scan(int v, int& total, int* words) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int upto = wave_inclusive_scan(v);
  __syncthreads();
  if (lane == 63) words[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < TABLE_THREADS / 64; ++w) {
    const int mine = words[w];
    if (w < wave) before += mine;
    total += mine;
  }
  return before + upto - v;
}

// The first workgroup: which rows need a page of their own, the free pages, who gets which, and the columns of the table
// that it decides: of a living row the last one that its tokens take and the reserved ones. The others bring the rest.
__global__ __launch_bounds__(TABLE_THREADS) void fork_assign_kernel(ForkArgs a) {
  __shared__ __attribute__((aligned(16))) int32_t tails[FORK_MAX_B];  // to a multiple of four, -1 behind the last
  __shared__ int words[TABLE_THREADS / 64];
  __shared__ int64_t lacks[TABLE_THREADS / 64];
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int64_t at = (int64_t)(blockIdx.x - 1) * TABLE_THREADS + tid;
    if (at >= (int64_t)a.B * a.W) return;
    const int b = (int)(at / a.W), column = (int)(at - (int64_t)b * a.W);
    const ForkRow row(a, b);
    if (row.parent >= 0 && column >= row.held - 1 && column < max(row.most, row.held)) return;
    if (row.parent < 0 || column >= row.held)
      a.table[at] = -1;
    else if (row.parent != b)
      a.table[at] = a.rows[at];
    return;
  }
  const int quads = (a.B + 3) / 4;
  for (int b = tid; b < 4 * quads; b += TABLE_THREADS) tails[b] = b < a.B ? a.tails[b] : -1;
  __syncthreads();
  // All but the lowest of the rows that share such a page take a copy; all, where others hold it too.
  uint32_t copies = 0;  // bit i: row tid + i * TABLE_THREADS
  int wanted = 0;
  int64_t over = 0;
  for (int b = tid, i = 0; b < a.B; b += TABLE_THREADS, ++i) {
    const int32_t tail = tails[b];
    bool copied = false;
    if (tail >= 0) {
      int same = 0;
      bool lowest = true;
#pragma unroll 4
      for (int q = 0; q < quads; ++q) {
        const int4 others = ((const int4*)tails)[q];
        const int equal = (others.x == tail ? 1 : 0) | (others.y == tail ? 2 : 0) | (others.z == tail ? 4 : 0) | (others.w == tail ? 8 : 0);
        same += __popc(equal);
        lowest = lowest && !(4 * q < b && (equal & ((1 << min(b - 4 * q, 4)) - 1)));
      }
      copied = !(lowest && load_count(a.counts + tail) == same);
    }
    copies |= copied ? 1u << i : 0u;
  }
  __syncthreads();
  for (int b = tid, i = 0; b < a.B; b += TABLE_THREADS, ++i)
    if (copies >> i & 1u) atomicSub(a.counts + tails[b], 1);
  __threadfence();
  // Pages wanted before each row.
  for (int base = 0, i = 0; base < a.B; base += TABLE_THREADS, ++i) {
    const int b = base + tid;
    if (b < a.B) {
      const ForkRow row(a, b);
      if (row.parent >= 0) {
        wanted += (copies >> i & 1u) + (int)max(min(row.most, (int64_t)a.W) - row.held, (int64_t)0);
        over += max(row.most - a.W, (int64_t)0);
      }
    }
  }
  int all;
  block_scan(wanted, all, words);
  // The first of the free pages, as many as are wanted.
  int found = 0;
  for (int base = 0; base < a.BLOCKS && found < all; base += TABLE_THREADS * 4) {
    int mine = 0;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int page = base + tid * 4 + i;
      if (page < a.BLOCKS && load_count(a.counts + page) == 0) {
        bits |= 1u << i;
        ++mine;
      }
    }
    int total;
    int at = found + block_scan(mine, total, words);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (bits >> i & 1u) {
        if (at < all) a.free_list[at] = base + tid * 4 + i;
        ++at;
      }
    found = min(found + total, all);
  }
  __syncthreads();
  int first = 0;
  int64_t lacking = over;
  for (int base = 0, i = 0; base < a.B; base += TABLE_THREADS, ++i) {
    const int b = base + tid;
    int mine = 0, copied = 0;
    int64_t held = 0, end = 0;
    if (b < a.B) {
      const ForkRow row(a, b);
      if (row.parent >= 0) {
        copied = copies >> i & 1u;
        held = row.held;
        end = max(min(row.most, (int64_t)a.W), held);
        mine = copied + (int)(end - held);
      }
    }
    int total;
    int at = first + block_scan(mine, total, words);
    first += total;
    if (b < a.B) {
      int32_t from = -1, to = -1;
      int32_t* const rows = a.table + (int64_t)b * a.W;
      const ForkRow row(a, b);
      auto take = [&](int64_t column) {
        const int32_t page = at < found ? a.free_list[at] : -1;
        ++at;
        rows[column] = page;
        if (page >= 0)
          a.counts[page] = 1;
        else
          ++lacking;
        return page;
      };
      if (copied) {
        to = take(held - 1);
        from = to >= 0 ? tails[b] : -1;
      } else if (row.parent >= 0 && row.parent != b && held > 0 && held <= a.W) {
        rows[held - 1] = a.rows[(int64_t)b * a.W + held - 1];
      }
      for (int64_t c = held; c < end; ++c) take(c);
      a.source[b] = from;
      a.destination[b] = to;
    }
  }
  // The number of pages that could not be had.
#pragma unroll
  for (int d = 1; d < 64; d *= 2) lacking += __shfl_xor((long long)lacking, d);
  __syncthreads();
  if ((tid & 63) == 0) lacks[tid >> 6] = lacking;
  __syncthreads();
  if (tid == 0) {
    int64_t sum = 0;
    for (int w = 0; w < TABLE_THREADS / 64; ++w) sum += lacks[w];
    *a.missing = (int32_t)min(sum, (int64_t)0x7fffffff);
  }
}

// ---- compaction ----------------------------------------------------------------

constexpr int SEGMENT = 256 * 16;  // pages of a workgroup

struct CompactArgs {
  int32_t* table;
  int32_t* counts;
  int32_t* source;
  int32_t* destination;
  int32_t* segments;  // workspace: pages in use of each segment
  int32_t* moves;     // workspace [BLOCKS]: of a page that moves, which move it is, else -1
  int64_t entries;    // of the table
  int32_t BLOCKS;
};
// Segments up to here are counted by every workgroup for itself, one launch less.
constexpr int FEW_SEGMENTS = 4;

__device__ __forceinline__ int sum_256(int v, int* words) {
  const int upto = wave_inclusive_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) words[threadIdx.x >> 6] = upto;
  __syncthreads();
  return words[0] + words[1] + words[2] + words[3];
}

__global__ __launch_bounds__(256) void compact_count_kernel(CompactArgs a) {
  __shared__ int words[4];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t page = (int64_t)blockIdx.x * SEGMENT + i * 256 + threadIdx.x;
    mine += page < a.BLOCKS && a.counts[page] > 0;
  }
  const int total = sum_256(mine, words);
  if (threadIdx.x == 0) a.segments[blockIdx.x] = total;
}

// With n pages in use, the k-th of those from n on moves to the k-th free one below n.
__global__ __launch_bounds__(256) void compact_moves_kernel(CompactArgs a, int segments) {
  __shared__ int words[4], step_sums[16][4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t base = (int64_t)blockIdx.x * SEGMENT;
  uint32_t bits = 0;  // bit i: page base + 256 i + tid is in use
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t page = base + i * 256 + tid;
    bits |= page < a.BLOCKS && a.counts[page] > 0 ? 1u << i : 0u;
  }
  int before = 0, all = 0, stays = 0;
  if (segments <= FEW_SEGMENTS) {
    for (int64_t i = tid; i < a.BLOCKS; i += 256) {
      const int v = a.counts[i] > 0;
      all += v;
      before += i < base ? v : 0;
    }
  } else {
    for (int i = tid; i < segments; i += 256) {
      const int v = a.segments[i];
      all += v;
      before += i < (int)blockIdx.x ? v : 0;
    }
  }
  const int n = sum_256(all, words);
  before = sum_256(before, words);
  // In use below n: the pages that stay.
  const int whole = segments <= FEW_SEGMENTS ? 0 : n / SEGMENT;
  for (int i = tid; i < whole; i += 256) stays += a.segments[i];
  for (int i = whole * SEGMENT + tid; i < n; i += 256) stays += a.counts[i] > 0;
  stays = sum_256(stays, words);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t wave_bits = __ballot(bits >> i & 1u);
    if (lane == 0) step_sums[i][wave] = __popcll(wave_bits);
  }
  __syncthreads();
  int used = before;  // pages in use ahead of these 256
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t page = base + i * 256 + tid;
    const bool in_use = bits >> i & 1u;
    int ahead = used + __popcll(__ballot(in_use) & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) ahead += step_sums[i][w];
      used += step_sums[i][w];
    }
    if (page < a.BLOCKS) {
      const int move = page >= n && in_use ? ahead - stays : -1;
      a.moves[page] = move;
      if (move >= 0) a.source[move] = (int)page;
      if (page < n && !in_use) a.destination[page - ahead] = (int)page;
    }
  }
  const int moves = n - stays;
  for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < a.BLOCKS / 2; i += (int64_t)gridDim.x * 256)
    if (i >= moves) {
      a.source[i] = -1;
      a.destination[i] = -1;
    }
}

// The table's entries, and the counts of the pages that moved.
__global__ __launch_bounds__(256) void compact_rename_kernel(CompactArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < a.entries) {
    const int32_t page = a.table[i];
    const int32_t move = names_page(page, a.BLOCKS) ? a.moves[page] : -1;
    if (move >= 0) a.table[i] = a.destination[move];
  }
  if (i < a.BLOCKS / 2) {
    const int from = a.source[i];
    if (from >= 0) {
      a.counts[a.destination[i]] = a.counts[from];
      a.counts[from] = 0;
    }
  }
}

namespace {

int power_shift(int32_t power) {
  int s = 0;
  while ((1 << s) < power) ++s;
  return s;
}

int check_fork(const ForkPagesParams* p) {
  if (!p) return AFA_E_NULL;
  if (p->B <= 0 || p->B > FORK_MAX_B || p->W <= 0 || p->BLOCKS <= 0 || p->BLOCKS > 1 << 28 || p->reserve < 0) return AFA_E_SHAPE;
  if (p->PAGE <= 0 || (p->PAGE & (p->PAGE - 1)) || p->W > 1 << 24 || (int64_t)p->B * p->W >= 1ll << 31) return AFA_E_SHAPE;
  return AFA_OK;
}

int check_compact(const CompactPagesParams* p) {
  if (!p) return AFA_E_NULL;
  if (p->B <= 0 || p->W <= 0 || p->BLOCKS <= 0 || p->BLOCKS > 1 << 28 || (int64_t)p->B * p->W > 1ll << 31) return AFA_E_SHAPE;
  return AFA_OK;
}

uint64_t rounded(uint64_t bytes) { return (bytes + 255) & ~(uint64_t)255; }

}  // namespace
}  // namespace afa

extern "C" int launch_copy_pages(void* stream, const void* const* caches, const uint64_t* page_bytes, int32_t n_caches,
                                 const int32_t* source, const int32_t* destination, int32_t pairs, int32_t BLOCKS) {
  using namespace afa;
  if (n_caches < 0 || pairs < 0 || BLOCKS <= 0) return AFA_E_SHAPE;
  if (n_caches == 0 || pairs == 0) return AFA_OK;
  if (!caches || !page_bytes || !source || !destination) return AFA_E_NULL;
  for (int32_t i = 0; i < n_caches; ++i) {  // of all caches before the first is written
    if (!caches[i]) return AFA_E_NULL;
    if (page_bytes[i] == 0 || page_bytes[i] > 1ull << 36) return AFA_E_SHAPE;
    // Far more than the list of a compaction takes: half as many pairs as a cache has pages.
    if ((page_bytes[i] + COPY_BYTES - 1) / COPY_BYTES * (uint64_t)pairs > 1ull << 32) return AFA_E_SHAPE;
  }
  hipStream_t s = (hipStream_t)stream;
  for (int32_t first = 0; first < n_caches; first += COPY_CACHES) {
    const int n = std::min(n_caches - first, COPY_CACHES);
    CopyArgs a;
    a.blocks = BLOCKS;
    uint64_t most = 0;
    for (int i = 0; i < n; ++i) {
      a.cache[i] = (uint8_t*)caches[first + i];
      a.bytes[i] = page_bytes[first + i];
      most = std::max(most, a.bytes[i]);
    }
    const uint64_t parts = (most + COPY_BYTES - 1) / COPY_BYTES;
    a.parts = (int32_t)parts;
    const int64_t each = (int64_t)(0xffffffffull / 256 / parts);  // pairs of a launch, which counts its threads in 32 bits
    for (int64_t at = 0; at < pairs; at += each) {
      a.source = source + at;
      a.destination = destination + at;
      const uint64_t groups = parts * (uint64_t)std::min<int64_t>(each, pairs - at);
      hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)groups, (unsigned)n), dim3(256), 0, s, a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
    }
  }
  return AFA_OK;
}

extern "C" int workspace_size_fork_pages(uint64_t* bytes, const ForkPagesParams* p) {
  using namespace afa;
  if (!bytes) return AFA_E_NULL;
  const int status = check_fork(p);
  if (status) return status;
  *bytes = rounded(4ull * p->B * p->W) + rounded(4ull * p->BLOCKS) + rounded(4ull * p->B);
  return AFA_OK;
}

extern "C" int launch_fork_pages(void* stream, int32_t* block_table, int32_t* page_counts, const int32_t* parents,
                                 const int32_t* seqused_kv, int32_t* source, int32_t* destination, int32_t* missing,
                                 void* workspace, uint64_t workspace_bytes, const ForkPagesParams* p) {
  using namespace afa;
  uint64_t need = 0;
  const int status = workspace_size_fork_pages(&need, p);
  if (status) return status;
  if (!block_table || !page_counts || !parents || !seqused_kv || !source || !destination || !missing) return AFA_E_NULL;
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return AFA_E_WORKSPACE;
  ForkArgs a;
  a.table = block_table;
  a.counts = page_counts;
  a.parents = parents;
  a.used = seqused_kv;
  a.source = source;
  a.destination = destination;
  a.missing = missing;
  a.rows = (int32_t*)workspace;
  a.free_list = (int32_t*)((uint8_t*)workspace + rounded(4ull * p->B * p->W));
  a.tails = (int32_t*)((uint8_t*)a.free_list + rounded(4ull * p->BLOCKS));
  a.B = p->B;
  a.W = p->W;
  a.BLOCKS = p->BLOCKS;
  a.page_shift = power_shift(p->PAGE);
  a.reserve = p->reserve;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(fork_rows_kernel, dim3((unsigned)((a.W + 255) / 256), (unsigned)a.B), dim3(256), 0, s, a);
  const int64_t others = ((int64_t)a.B * a.W + TABLE_THREADS - 1) / TABLE_THREADS;
  hipLaunchKernelGGL(fork_assign_kernel, dim3((unsigned)(1 + others)), dim3(TABLE_THREADS), 0, s, a);
  return (int)hipGetLastError();
}

extern "C" int workspace_size_compact_pages(uint64_t* bytes, const CompactPagesParams* p) {
  using namespace afa;
  if (!bytes) return AFA_E_NULL;
  const int status = check_compact(p);
  if (status) return status;
  const uint64_t segments = ((uint64_t)p->BLOCKS + SEGMENT - 1) / SEGMENT;
  *bytes = rounded(4 * segments) + rounded(4ull * p->BLOCKS);
  return AFA_OK;
}

extern "C" int launch_compact_pages(void* stream, int32_t* block_table, int32_t* page_counts, int32_t* source,
                                    int32_t* destination, void* workspace, uint64_t workspace_bytes,
                                    const CompactPagesParams* p) {
  using namespace afa;
  uint64_t need = 0;
  const int status = workspace_size_compact_pages(&need, p);
  if (status) return status;
  if (!block_table || !page_counts || (p->BLOCKS > 1 && (!source || !destination))) return AFA_E_NULL;
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return AFA_E_WORKSPACE;
  if (p->BLOCKS == 1) return AFA_OK;
  const int segments = (p->BLOCKS + SEGMENT - 1) / SEGMENT;
  CompactArgs a;
  a.table = block_table;
  a.counts = page_counts;
  a.source = source;
  a.destination = destination;
  a.segments = (int32_t*)workspace;
  a.moves = (int32_t*)((uint8_t*)workspace + rounded(4ull * segments));
  a.entries = (int64_t)p->B * p->W;
  a.BLOCKS = p->BLOCKS;
  hipStream_t s = (hipStream_t)stream;
  if (segments > FEW_SEGMENTS) hipLaunchKernelGGL(compact_count_kernel, dim3((unsigned)segments), dim3(256), 0, s, a);
  hipLaunchKernelGGL(compact_moves_kernel, dim3((unsigned)segments), dim3(256), 0, s, a, segments);
  const int64_t items = std::max<int64_t>(a.entries, a.BLOCKS / 2);
  hipLaunchKernelGGL(compact_rename_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
