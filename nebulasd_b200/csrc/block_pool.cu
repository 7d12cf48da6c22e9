// Blocks of the paged KV cache copied, forked, freed and compacted on the device.
//
// The pool is the callers': caches [num_blocks][layers * kv heads][block_size][head_dim], a block table
// [rows][max_blocks] with the first seq_blocks[row] entries of a row in use, and one reference count per
// block (0: free).  Every operator reads its lists on the device, so that a program which
// chooses its branches on the device never waits for the host, and leaves the same result whatever the
// order of its threads: blocks are taken lowest first, counts change by integer atomics.
//
// The simple form: plans by one CTA, copies with 16-byte loads and stores.
#include "neb_common.cuh"

namespace neb {
namespace blocks {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;

struct Caches {
  char* plane[2];
  long long num_blocks;
  int tiles;        // layers * kv heads
  int block_size;   // tokens
  int token_bytes;  // of one tile (a multiple of 16)
};

struct Tables {
  int32_t* table;
  int rows, width;
  int32_t* seq_blocks;
  int32_t* refs;
};

__device__ __forceinline__ void report(unsigned int* bits, unsigned int bit) {
  if (bits) atomicOr(bits, bit);
}

// Exclusive prefix sum over the block's threads; `total` gets the sum.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < warps; ++i) {
    const int s = warp_sums[i];
    before += i < warp ? s : 0;
    all += s;
  }
  total = all;
  return before + v - x;
}

// Copies the first `tokens` tokens of every tile of [t0, t1) of one block and plane, by one CTA.
__device__ __forceinline__ void copy_tiles(const Caches& c, int plane, long long src, long long dst, int tokens, int t0,
                                           int t1) {
  const int words = c.token_bytes / 16, pitch = c.block_size * words, live = tokens * words;
  const long long block_words = (long long)c.tiles * pitch;
  const uint4* s = reinterpret_cast<const uint4*>(c.plane[plane]) + src * block_words + (long long)t0 * pitch;
  uint4* d = reinterpret_cast<uint4*>(c.plane[plane]) + dst * block_words + (long long)t0 * pitch;
  const int n = (t1 - t0) * live;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int t = i / live;
    const long long at = (long long)t * pitch + (i - t * live);
    __stcs(d + at, __ldcs(s + at));
  }
}

// ------------------------------------------------------------------------ copy
struct CopyParams {
  Caches c;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;  // or null: whole blocks
  int n;
  int chunk_tiles, chunks;  // tiles per work item, items per block and plane
  unsigned int* error_bits;
};

// One pair's checks, by the whole CTA: out of range, or in conflict with another pair.
__device__ __forceinline__ bool pair_ok(const CopyParams& p, int i, int& src, int& dst, int& tokens) {
  src = p.src[i];
  dst = p.dst[i];
  tokens = p.tokens ? p.tokens[i] : p.c.block_size;
  unsigned int bad = 0;
  if (src < 0 || src >= p.c.num_blocks || dst < 0 || dst >= p.c.num_blocks) bad |= kErrBlockIndex;
  if (tokens < 0 || tokens > p.c.block_size) bad |= kErrInvalidRows;
  bool clash = false;
  for (int j = threadIdx.x; j < p.n; j += blockDim.x) {
    const int other = p.dst[j];
    clash |= j != i && (other == dst || other == src);
  }
  if (__syncthreads_or(clash)) bad |= kErrCopyConflict;
  if (bad && threadIdx.x == 0) report(p.error_bits, bad);
  return bad == 0 && src != dst;
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const CopyParams p) {
  const long long items = 2ll * p.n * p.chunks;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int chunk = (int)(it % p.chunks);
    const long long rest = it / p.chunks;
    const int plane = (int)(rest & 1), pair = (int)(rest >> 1);
    int src, dst, tokens;
    if (!pair_ok(p, pair, src, dst, tokens)) continue;
    const int t0 = chunk * p.chunk_tiles;
    copy_tiles(p.c, plane, src, dst, tokens, t0, min(p.c.tiles, t0 + p.chunk_tiles));
  }
}

// ------------------------------------------------------------------------ fork
struct ForkParams {
  Caches c;
  Tables t;
  const int32_t* parents;
  const int32_t* children;
  const int32_t* lens;
  const int32_t* capacities;  // or null
  int n;
  int32_t* plan;   // [n][4]: shared blocks, all blocks (-1: refused), first of its slots, partial tokens
  int32_t* slots;  // free blocks, lowest first
  unsigned int* error_bits;
  int chunk_tiles, chunks;
};

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const ForkParams p) {
  __shared__ int sums[kPlanThreads / 32];
  const int tid = threadIdx.x, bs = p.c.block_size;
  // Each child's shape; nothing is written to the pool yet, so a row that is another child's parent is
  // read as it was.
  for (int i = tid; i < p.n; i += kPlanThreads) {
    const int parent = p.parents[i], child = p.children[i], len = p.lens[i];
    const int cap = max(len, p.capacities ? p.capacities[i] : 0);
    unsigned int bad = 0;
    if (child < 0 || child >= p.t.rows || (len > 0 && (parent < 0 || parent >= p.t.rows))) bad |= kErrSeqId;
    if (len < 0 || (p.capacities && p.capacities[i] < 0)) bad |= kErrInvalidRows;
    const int shared = max(len, 0) / bs;
    const int total = (int)(((long long)max(cap, 0) + bs - 1) / bs);
    if (total > p.t.width) bad |= kErrTooManyBlocks;
    if (!bad) {
      if (p.t.seq_blocks[child] != 0) bad |= kErrInvalidRows;
      if (len > 0 && ((long long)len + bs - 1) / bs > p.t.seq_blocks[parent]) bad |= kErrInvalidRows;
    }
    if (bad) report(p.error_bits, bad);
    p.plan[4 * i] = shared;
    p.plan[4 * i + 1] = bad ? -1 : total;
    p.plan[4 * i + 3] = max(len, 0) - shared * bs;
  }
  __syncthreads();
  // A row listed twice goes to its first child: the lowest claim wins.
  for (int i = tid; i < p.n; i += kPlanThreads)
    if (p.plan[4 * i + 1] >= 0) atomicMin(&p.t.seq_blocks[p.children[i]], i - p.n);
  __syncthreads();
  for (int i = tid; i < p.n; i += kPlanThreads)
    if (p.plan[4 * i + 1] >= 0 && __ldcg(&p.t.seq_blocks[p.children[i]]) != i - p.n) {
      report(p.error_bits, kErrInvalidRows);
      p.plan[4 * i + 1] = -1;
    }
  __syncthreads();
  // Slots in the children's order.
  int need = 0;
  for (int base = 0; base < p.n; base += kPlanThreads) {
    const int i = base + tid;
    const int mine = i < p.n && p.plan[4 * i + 1] >= 0 ? p.plan[4 * i + 1] - p.plan[4 * i] : 0;
    int all;
    const int before = block_scan(mine, sums, all);
    if (i < p.n) p.plan[4 * i + 2] = need + before;
    need += all;
  }
  // The lowest free blocks.
  int found = 0;
  for (long long base = 0; base < p.c.num_blocks && found < need; base += kPlanThreads) {
    const long long b = base + tid;
    const int is_free = b < p.c.num_blocks && p.t.refs[b] == 0;
    int all;
    const int at = found + block_scan(is_free, sums, all);
    if (is_free && at < need) p.slots[at] = (int)b;
    found += all;
  }
  for (int i = tid; i < p.n; i += kPlanThreads) {
    const int total = p.plan[4 * i + 1];
    if (total < 0) continue;
    const int mine = total - p.plan[4 * i];
    const bool granted = mine == 0 || p.plan[4 * i + 2] + mine <= found;
    if (!granted) {
      report(p.error_bits, kErrNoFreeBlock);
      p.plan[4 * i + 1] = -1;
    }
    p.t.seq_blocks[p.children[i]] = granted ? total : 0;
  }
}

__global__ void __launch_bounds__(kCopyThreads) fork_kernel(const ForkParams p) {
  const long long items = 2ll * p.n * p.chunks;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int chunk = (int)(it % p.chunks);
    const long long rest = it / p.chunks;
    const int plane = (int)(rest & 1), i = (int)(rest >> 1);
    const int shared = p.plan[4 * i], total = p.plan[4 * i + 1], slot = p.plan[4 * i + 2], part = p.plan[4 * i + 3];
    if (total < 0) continue;
    const int32_t* from = p.t.table + (long long)p.parents[i] * p.t.width;
    if (chunk == 0 && plane == 0) {
      int32_t* to = p.t.table + (long long)p.children[i] * p.t.width;
      for (int j = threadIdx.x; j < total; j += blockDim.x) {
        int b;
        if (j < shared) {
          b = from[j];
          if (b < 0 || b >= p.c.num_blocks) {
            report(p.error_bits, kErrBlockIndex);
            b = -1;
          } else if (atomicAdd(&p.t.refs[b], 1) <= 0) {
            report(p.error_bits, kErrRefCount);
          }
        } else {
          b = p.slots[slot + j - shared];
          p.t.refs[b] = 1;
        }
        to[j] = b;
      }
    }
    if (part > 0) {
      const int src = from[shared];
      if (src < 0 || src >= p.c.num_blocks) {
        if (threadIdx.x == 0) report(p.error_bits, kErrBlockIndex);
        continue;
      }
      const int t0 = chunk * p.chunk_tiles;
      copy_tiles(p.c, plane, src, p.slots[slot], part, t0, min(p.c.tiles, t0 + p.chunk_tiles));
    }
  }
}

// ------------------------------------------------------------------------ free
struct FreeParams {
  Tables t;
  long long num_blocks;
  const int32_t* list;
  int n;
  unsigned int* error_bits;
};

__global__ void __launch_bounds__(kCopyThreads) free_kernel(const FreeParams p) {
  __shared__ int held;
  for (int i = blockIdx.x; i < p.n; i += gridDim.x) {
    const int row = p.list[i];
    if (row < 0 || row >= p.t.rows) {
      if (threadIdx.x == 0) report(p.error_bits, kErrSeqId);
      continue;
    }
    __syncthreads();
    // Whoever takes the count frees the row: one that is listed twice is freed once.
    if (threadIdx.x == 0) {
      held = atomicExch(&p.t.seq_blocks[row], 0);
      if (held < 0 || held > p.t.width) {
        report(p.error_bits, kErrTooManyBlocks);
        held = held < 0 ? 0 : p.t.width;
      }
    }
    __syncthreads();
    int32_t* entry = p.t.table + (long long)row * p.t.width;
    for (int j = threadIdx.x; j < held; j += blockDim.x) {
      const int b = entry[j];
      entry[j] = -1;
      if (b < 0 || b >= p.num_blocks) {
        report(p.error_bits, kErrBlockIndex);
      } else if (atomicSub(&p.t.refs[b], 1) <= 0) {
        atomicAdd(&p.t.refs[b], 1);  // it was free already: a count never stays negative
        report(p.error_bits, kErrRefCount);
      }
    }
  }
}

// --------------------------------------------------------------------- compact
struct CompactParams {
  Caches c;
  Tables t;
  int32_t* new_index;
  int32_t* header;  // number of moves
  int32_t* src;
  int32_t* dst;
  unsigned int* error_bits;
  int chunk_tiles, chunks;
};

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactParams p) {
  __shared__ int sums[kPlanThreads / 32];
  const int tid = threadIdx.x;
  const long long nb = p.c.num_blocks;
  int mine = 0;
  for (long long b = tid; b < nb; b += kPlanThreads) mine += p.t.refs[b] > 0;
  int live;
  block_scan(mine, sums, live);
  // The i-th free block below `live` takes the i-th live block at or above it.
  int holes = 0, movers = 0;
  for (long long base = 0; base < nb; base += kPlanThreads) {
    const long long b = base + tid;
    const bool in = b < nb, used = in && p.t.refs[b] > 0;
    const bool hole = in && !used && b < live, mover = used && b >= live;
    int all_holes, all_movers;
    const int ah = block_scan(hole, sums, all_holes), am = block_scan(mover, sums, all_movers);
    if (hole) p.dst[holes + ah] = (int)b;
    if (mover) p.src[movers + am] = (int)b;
    if (in) p.new_index[b] = used ? (int)b : -1;
    holes += all_holes;
    movers += all_movers;
  }
  __syncthreads();
  for (int i = tid; i < movers; i += kPlanThreads) {
    const int s = p.src[i], d = p.dst[i];
    p.new_index[s] = d;
    p.t.refs[d] = p.t.refs[s];
    p.t.refs[s] = 0;
  }
  if (tid == 0) p.header[0] = movers;
}

__global__ void __launch_bounds__(kCopyThreads) compact_kernel(const CompactParams p) {
  // Table entries follow their blocks.
  const long long entries = (long long)p.t.rows * p.t.width;
  for (long long e = blockIdx.x * (long long)blockDim.x + threadIdx.x; e < entries;
       e += (long long)gridDim.x * blockDim.x) {
    const int row = (int)(e / p.t.width);
    if (e - (long long)row * p.t.width >= p.t.seq_blocks[row]) continue;
    const int b = p.t.table[e];
    if (b < 0 || b >= p.c.num_blocks) {
      report(p.error_bits, kErrBlockIndex);
      continue;
    }
    const int to = p.new_index[b];
    if (to < 0) report(p.error_bits, kErrRefCount);
    if (to != b) p.t.table[e] = to;
  }
  const long long items = 2ll * p.header[0] * p.chunks;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int chunk = (int)(it % p.chunks);
    const long long rest = it / p.chunks;
    const int plane = (int)(rest & 1), i = (int)(rest >> 1), t0 = chunk * p.chunk_tiles;
    copy_tiles(p.c, plane, p.src[i], p.dst[i], p.c.block_size, t0, min(p.c.tiles, t0 + p.chunk_tiles));
  }
}

// ------------------------------------------------------------------------ host
constexpr int kChunkBytes = 64 * 1024;

static int fill_caches(Caches& c, void* k, void* v, int64_t num_blocks, int32_t tiles, int32_t block_size,
                       int32_t token_bytes) {
  NEB_REQUIRE(num_blocks > 0 && num_blocks <= INT_MAX && tiles > 0 && block_size > 0, NEB_ERR_INVALID,
              "num_blocks, tiles_per_block and block_size must be positive (num_blocks below 2^31)");
  NEB_REQUIRE(token_bytes > 0 && token_bytes % 16 == 0, NEB_ERR_UNSUPPORTED,
              "token_bytes must be a positive multiple of 16 (got %d)", token_bytes);
  NEB_REQUIRE((long long)tiles * block_size * token_bytes < (1ll << 31), NEB_ERR_UNSUPPORTED,
              "a block of 2 GiB or more per plane is not supported");
  NEB_REQUIRE(k && v, NEB_ERR_INVALID, "null cache");
  NEB_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0, NEB_ERR_INVALID,
              "caches must be 16-byte aligned");
  c.plane[0] = static_cast<char*>(k);
  c.plane[1] = static_cast<char*>(v);
  c.num_blocks = num_blocks;
  c.tiles = tiles;
  c.block_size = block_size;
  c.token_bytes = token_bytes;
  return NEB_OK;
}

static int fill_tables(Tables& t, int32_t* table, int32_t rows, int32_t width, int32_t* seq_blocks, int32_t* refs) {
  NEB_REQUIRE(rows > 0 && width > 0, NEB_ERR_INVALID, "block_table_rows and max_blocks_per_seq must be positive");
  NEB_REQUIRE((long long)rows * width < (1ll << 31), NEB_ERR_UNSUPPORTED, "a block table of 2^31 entries or more");
  NEB_REQUIRE(table && seq_blocks && refs, NEB_ERR_INVALID, "null table");
  t.table = table;
  t.rows = rows;
  t.width = width;
  t.seq_blocks = seq_blocks;
  t.refs = refs;
  return NEB_OK;
}

static void cut(const Caches& c, int& chunk_tiles, int& chunks) {
  const int tile_bytes = c.block_size * c.token_bytes;
  chunk_tiles = kChunkBytes / tile_bytes > 0 ? kChunkBytes / tile_bytes : 1;
  chunks = (c.tiles + chunk_tiles - 1) / chunk_tiles;
}

static int copy_grid(long long items, unsigned& grid) {
  int dev = 0;
  NEB_CUDA(cudaGetDevice(&dev));
  const long long most = 8ll * num_sms(dev);
  NEB_REQUIRE(most > 0, NEB_ERR_CUDA, "could not size the grid for device %d", dev);
  grid = (unsigned)(items < most ? (items > 0 ? items : 1) : most);
  return NEB_OK;
}

}  // namespace blocks
}  // namespace neb

using namespace neb;
using namespace neb::blocks;

extern "C" {

int neb_copy_blocks(void* k_cache, void* v_cache, int64_t num_blocks, int32_t tiles_per_block, int32_t block_size,
                    int32_t token_bytes, const int32_t* src, const int32_t* dst, const int32_t* num_tokens,
                    int32_t num_pairs, uint32_t* error_bits, void* stream) {
  CopyParams p;
  if (int rc = fill_caches(p.c, k_cache, v_cache, num_blocks, tiles_per_block, block_size, token_bytes)) return rc;
  NEB_REQUIRE(num_pairs >= 0, NEB_ERR_INVALID, "negative number of pairs");
  if (num_pairs == 0) return NEB_OK;
  NEB_REQUIRE(src && dst, NEB_ERR_INVALID, "null block list");
  p.src = src;
  p.dst = dst;
  p.tokens = num_tokens;
  p.n = num_pairs;
  p.error_bits = error_bits;
  cut(p.c, p.chunk_tiles, p.chunks);
  unsigned grid;
  if (int rc = copy_grid(2ll * num_pairs * p.chunks, grid)) return rc;
  copy_kernel<<<grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  NEB_CUDA(cudaGetLastError());
  return NEB_OK;
}

size_t neb_fork_workspace_bytes(int64_t num_blocks, int32_t num_children) {
  if (num_blocks <= 0 || num_blocks > INT_MAX || num_children < 0) return 0;
  return 16 * (size_t)num_children + 4 * (size_t)num_blocks;
}

int neb_fork_sequences(void* k_cache, void* v_cache, int64_t num_blocks, int32_t tiles_per_block, int32_t block_size,
                       int32_t token_bytes, int32_t* block_table, int32_t block_table_rows,
                       int32_t max_blocks_per_seq, int32_t* seq_blocks, int32_t* ref_counts, const int32_t* parents,
                       const int32_t* children, const int32_t* seq_lens, const int32_t* capacities,
                       int32_t num_children, void* workspace, size_t workspace_bytes, uint32_t* error_bits,
                       void* stream) {
  ForkParams p;
  if (int rc = fill_caches(p.c, k_cache, v_cache, num_blocks, tiles_per_block, block_size, token_bytes)) return rc;
  if (int rc = fill_tables(p.t, block_table, block_table_rows, max_blocks_per_seq, seq_blocks, ref_counts)) return rc;
  NEB_REQUIRE(num_children >= 0, NEB_ERR_INVALID, "negative number of children");
  if (num_children == 0) return NEB_OK;
  NEB_REQUIRE(parents && children && seq_lens, NEB_ERR_INVALID, "null sequence list");
  NEB_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0 &&
                  workspace_bytes >= neb_fork_workspace_bytes(num_blocks, num_children),
              NEB_ERR_WORKSPACE, "workspace missing, misaligned or smaller than the %zu bytes required",
              neb_fork_workspace_bytes(num_blocks, num_children));
  p.parents = parents;
  p.children = children;
  p.lens = seq_lens;
  p.capacities = capacities;
  p.n = num_children;
  p.plan = static_cast<int32_t*>(workspace);
  p.slots = p.plan + 4ll * num_children;
  p.error_bits = error_bits;
  cut(p.c, p.chunk_tiles, p.chunks);
  unsigned grid;
  if (int rc = copy_grid(2ll * num_children * p.chunks, grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  fork_plan_kernel<<<1, kPlanThreads, 0, s>>>(p);
  NEB_CUDA(cudaGetLastError());
  fork_kernel<<<grid, kCopyThreads, 0, s>>>(p);
  NEB_CUDA(cudaGetLastError());
  return NEB_OK;
}

int neb_free_sequences(int32_t* block_table, int32_t block_table_rows, int32_t max_blocks_per_seq,
                       int32_t* seq_blocks, int32_t* ref_counts, int64_t num_blocks, const int32_t* rows,
                       int32_t num_rows, uint32_t* error_bits, void* stream) {
  FreeParams p;
  if (int rc = fill_tables(p.t, block_table, block_table_rows, max_blocks_per_seq, seq_blocks, ref_counts)) return rc;
  NEB_REQUIRE(num_blocks > 0 && num_blocks <= INT_MAX, NEB_ERR_INVALID, "num_blocks must be in [1, 2^31)");
  NEB_REQUIRE(num_rows >= 0, NEB_ERR_INVALID, "negative number of rows");
  if (num_rows == 0) return NEB_OK;
  NEB_REQUIRE(rows, NEB_ERR_INVALID, "null row list");
  p.num_blocks = num_blocks;
  p.list = rows;
  p.n = num_rows;
  p.error_bits = error_bits;
  unsigned grid;
  if (int rc = copy_grid(num_rows, grid)) return rc;
  free_kernel<<<grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  NEB_CUDA(cudaGetLastError());
  return NEB_OK;
}

size_t neb_compact_workspace_bytes(int64_t num_blocks) {
  if (num_blocks <= 0 || num_blocks > INT_MAX) return 0;
  return 16 + 8 * ((size_t)num_blocks / 2 + 1);
}

int neb_compact_blocks(void* k_cache, void* v_cache, int64_t num_blocks, int32_t tiles_per_block, int32_t block_size,
                       int32_t token_bytes, int32_t* block_table, int32_t block_table_rows,
                       int32_t max_blocks_per_seq, int32_t* seq_blocks, int32_t* ref_counts, int32_t* new_index,
                       void* workspace, size_t workspace_bytes, uint32_t* error_bits, void* stream) {
  CompactParams p;
  if (int rc = fill_caches(p.c, k_cache, v_cache, num_blocks, tiles_per_block, block_size, token_bytes)) return rc;
  if (int rc = fill_tables(p.t, block_table, block_table_rows, max_blocks_per_seq, seq_blocks, ref_counts)) return rc;
  NEB_REQUIRE(new_index, NEB_ERR_INVALID, "new_index is null");
  NEB_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0 &&
                  workspace_bytes >= neb_compact_workspace_bytes(num_blocks),
              NEB_ERR_WORKSPACE, "workspace missing, misaligned or smaller than the %zu bytes required",
              neb_compact_workspace_bytes(num_blocks));
  p.new_index = new_index;
  p.header = static_cast<int32_t*>(workspace);
  p.src = p.header + 4;
  p.dst = p.src + (num_blocks / 2 + 1);
  p.error_bits = error_bits;
  cut(p.c, p.chunk_tiles, p.chunks);
  unsigned grid;
  if (int rc = copy_grid((num_blocks / 2 + 1) * 2ll * p.chunks, grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(p);
  NEB_CUDA(cudaGetLastError());
  compact_kernel<<<grid, kCopyThreads, 0, s>>>(p);
  NEB_CUDA(cudaGetLastError());
  return NEB_OK;
}

}  // extern "C"
