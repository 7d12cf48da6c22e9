// Blocks of the paged KV cache copied, forked, freed and compacted on the device.
//
// The pool is the callers': caches [num_blocks][layers * kv heads][block_size][head_dim], a block table
// [rows][max_blocks] with the first seq_blocks[row] entries of a row in use, and one reference count per
// block (0: free).  Every operator reads its lists on the device, so that a program which chooses its
// branches on the device never waits for the host, and leaves the same result whatever the order of its
// threads: blocks are taken lowest first, counts change by integer atomics.
//
// Fork and compact are two launches.  The plan is one thread-block cluster: its eight CTAs turn the
// reference counts into a bitmap in shared memory, exchange their sums over distributed shared memory and so
// give every free (or moved) block its rank without a grid-wide wait.  The second launch, which programmatic
// serialisation brings up meanwhile, spreads tables and copies over the GPU.  A copy is bound by HBM (every byte
// read and written once): a warp moves a 4 KB tile (one layer and head) at a time with up to eight 16-byte loads
// per lane before the first store.
#include "neb_common.cuh"
#include "sm100.cuh"

namespace neb {
namespace blocks {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanCtas = 8;                       // one cluster
constexpr int kMapCtas = kPlanCtas - 1;            // of a fork's plan: the first CTA has the children
constexpr long long kMaxPoolBlocks = 8ll << 20;    // a plan CTA's bitmap: 147 KB at most
constexpr int kCopyThreads = 256;
constexpr int kCopyWarps = kCopyThreads / 32;
constexpr int kLoads = 8;                          // 16-byte loads per lane in flight
// Copies of whole blocks run two CTAs per SM: 64 KB of loads in flight per SM, then as many stores (more, and
// reads and writes alternate in shorter runs: 512 blocks of 1.2 MB per plane in items of 64 KB 392 us, with four
// CTAs 415 us, with one 519 us).  Items of 128 KB copy scattered pairs best (383 us, 6.3 TB/s; 64 KB 395, 32 KB
// 420), items of 32 KB the ascending ones of a compaction (2.4 GB moved, 768 us; 64 KB 777, 128 KB 786).  Items are
// counted in tiles; these sizes are those of 4 KB tiles (16 tokens of 128 fp16).  Partial blocks have half the loads
// in flight per warp: four CTAs, items of one tile per warp (64 partial blocks of 28 layers 24 us, 5.2 TB/s; with two
// CTAs 27 us, with two tiles per warp 25 us).
constexpr int kWholeCtas = 2, kWholeTiles = 4 * kCopyWarps, kMoveTiles = kCopyWarps;
constexpr int kPartCtas = 4, kPartTiles = kCopyWarps;

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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  const int sum = warp_sums[lane];  // kPlanWarps == 32
  total = __reduce_add_sync(~0u, sum);
  return __reduce_add_sync(~0u, lane < warp ? sum : 0) + v - x;
}
static_assert(kPlanWarps == 32, "block_scan reads one sum per lane");

// ---------------------------------------------------------------------- copies
// The first `live` of a tile's 16-byte words.
__device__ __forceinline__ void copy_tile(const uint4* s, uint4* d, int live) {
  const int lane = threadIdx.x & 31;
  for (int base = lane; base < live; base += 32 * kLoads) {
    uint4 v[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (base + 32 * u < live) v[u] = ld_stream_v4(s + base + 32 * u);
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (base + 32 * u < live) __stcs(d + base + 32 * u, v[u]);
  }
}

struct Pair {
  int src, dst, tokens;
};

// Copies all pairs' tiles, K plane before V plane, in items of kTiles tiles of one block and plane that go round
// the CTAs, a tile per warp: what the GPU reads and writes at a time stays a few tens of MB of neighbouring
// tiles.  (A range of tiles per warp instead: 2 to 6 % slower.)  load(i) fetches a pair, for the next item before
// this one is copied (3 % of a compaction; a fork's pair beyond its first 256 is two loads that depend on each
// other, and they are waited for); keep(i, pair), called by the whole CTA, says whether it is copied.
template <int kTiles, typename Load, typename Keep>
__device__ __forceinline__ void copy_pairs(const Caches& c, int pairs, Load load, Keep keep) {
  const int words = c.token_bytes / 16, pitch = c.block_size * words, chunks = (c.tiles + kTiles - 1) / kTiles;
  const long long items = 2ll * pairs * chunks;
  long long it = blockIdx.x;
  if (it >= items) return;
  Pair next = load((int)(it / chunks >> 1));
  while (it < items) {
    const Pair pair = next;
    const long long plane_no = it / chunks;
    const int tile = (int)(it - plane_no * chunks) * kTiles, plane = (int)(plane_no & 1);
    it += gridDim.x;
    if (it < items) next = load((int)(it / chunks >> 1));
    if (!keep((int)(plane_no >> 1), pair)) continue;
    const int n = min(kTiles, c.tiles - tile), live = pair.tokens * words;
    const uint4* s = reinterpret_cast<const uint4*>(c.plane[plane]) + ((long long)pair.src * c.tiles + tile) * pitch;
    uint4* d = reinterpret_cast<uint4*>(c.plane[plane]) + ((long long)pair.dst * c.tiles + tile) * pitch;
    for (int t = threadIdx.x >> 5; t < n; t += kCopyWarps)
      copy_tile(s + (long long)t * pitch, d + (long long)t * pitch, live);
  }
}

// ------------------------------------------------------------------------ copy
struct CopyParams {
  Caches c;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;  // or null: whole blocks
  int n;
  unsigned int* error_bits;
};

// Every item compares its pair with all destinations: one comparison per thread up to 256 pairs, and from there on
// reads of the list that grow with the square of the pairs.  Of 36-layer blocks 4,096 pairs copy at 6.5 TB/s and
// 16,384 at 5.9; of one-layer ones 4,096 at 4.8, 16,384 at 3.3 and 32,768 at 1.9.
template <int kCtas, int kTiles>
__global__ void __launch_bounds__(kCopyThreads, kCtas) copy_kernel(const __grid_constant__ CopyParams p) {
  const int own = (int)threadIdx.x < p.n ? p.dst[threadIdx.x] : -1;  // the thread's share of the first destinations
  copy_pairs<kTiles>(
      p.c, p.n,
      [&](int i) { return Pair{p.src[i], p.dst[i], p.tokens ? p.tokens[i] : p.c.block_size}; },
      [&](int i, const Pair& a) {
        unsigned int bad = 0;
        if (a.src < 0 || a.src >= p.c.num_blocks || a.dst < 0 || a.dst >= p.c.num_blocks) bad |= kErrBlockIndex;
        if (a.tokens < 0 || a.tokens > p.c.block_size) bad |= kErrInvalidRows;
        bool clash = (int)threadIdx.x < p.n && (int)threadIdx.x != i && (own == a.dst || own == a.src);
        for (int j = threadIdx.x + kCopyThreads; j < p.n; j += kCopyThreads) {
          const int other = p.dst[j];
          clash |= j != i && (other == a.dst || other == a.src);
        }
        if (__syncthreads_or(clash)) bad |= kErrCopyConflict;
        if (bad && threadIdx.x == 0) report(p.error_bits, bad);
        return bad == 0 && a.src != a.dst;
      });
}

// ------------------------------------------------------------------------ plans
// A plan CTA's part of the pool: blocks [first, first + count), a bit for each in `map`.
struct PlanShared {
  int sums[kPlanWarps];
  int cta_bits[kPlanCtas];  // of every CTA of the cluster
  int cta_more[kPlanCtas];
  unsigned int map[1];      // (dynamic)
};
struct PlanPart {
  long long first;
  int count, words;
};
__device__ __forceinline__ PlanPart plan_part(long long num_blocks, int index, int parts) {
  const long long per = ((num_blocks + parts * 32 - 1) / (parts * 32)) * 32;
  PlanPart r;
  r.first = per * index;
  r.count = (int)max(0ll, min(per, num_blocks - r.first));
  r.words = (r.count + 31) / 32;
  return r;
}
static size_t plan_smem(long long num_blocks, int parts) {
  const long long per = ((num_blocks + parts * 32 - 1) / (parts * 32)) * 32;
  return sizeof(PlanShared) + 4 * (size_t)(per / 32);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// One int into every CTA's shared memory, at the place of this CTA.
__device__ __forceinline__ void cluster_share(int* slots, int value) {
  if (threadIdx.x < kPlanCtas) {
    uint32_t to;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(sm100::smem_u32(slots + blockIdx.x)), "r"(threadIdx.x));
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(value) : "memory");
  }
}

// Bits of the part's blocks whose count satisfies `bit`; returns how many (over the CTA).  The warp that has a word
// calls also(word, in, count) for its blocks.
template <typename Bit, typename Also>
__device__ __forceinline__ int build_map(PlanShared& sh, const PlanPart& part, const int32_t* refs, Bit bit,
                                         Also also) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kAhead = 16;  // words of a warp whose counts are loaded before the first is used
  int mine = 0;
  for (int w = warp; w < part.words; w += kAhead * kPlanWarps) {
    int r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = 32 * (w + u * kPlanWarps) + lane;
      r[u] = i < part.count ? refs[part.first + i] : 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = w + u * kPlanWarps;
      if (at >= part.words) break;
      const bool in = 32 * at + lane < part.count;
      const unsigned int word = __ballot_sync(~0u, in && bit(r[u]));
      also(at, in, r[u]);
      if (lane == 0) sh.map[at] = word;
      mine += __popc(word);
    }
  }
  int total;
  block_scan(lane == 0 ? mine : 0, sh.sums, total);
  return total;
}

// fn(i, before) for every set bit i of the part, `before` set bits of the part before it.
template <typename Fn>
__device__ __forceinline__ void each_bit(PlanShared& sh, int words, Fn fn) {
  int done = 0;
  for (int base = 0; base < words; base += kPlanThreads) {
    const int w = base + threadIdx.x;
    unsigned int left = w < words ? sh.map[w] : 0u;
    int all, before = block_scan(__popc(left), sh.sums, all);
    for (before += done; left; left &= left - 1) fn(32 * w + __ffs(left) - 1, before++);
    done += all;
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
  int32_t* plan;     // [n][4]: shared blocks, all blocks (-1: refused), first of its slots, partial tokens
  int32_t* partial;  // [n]: the partial tokens' block, or kNoBlock, kNoCount
  int32_t* slots;    // free blocks, lowest first
  unsigned int* uncounted;  // a bit per block: no positive count before the call
  unsigned int* error_bits;
};
constexpr int kNoBlock = -1, kNoCount = -2;  // an index out of range; a block without a positive count

// The children's shapes and their slots in order, by the first CTA, a child per thread and round: three round
// trips to memory for up to 1,024 children.  Returns the slots needed; `last` is the thread's child of the last
// round as written to p.plan.
__device__ __forceinline__ int plan_children(const ForkParams& p, int* sums, int4& last) {
  const int bs = p.c.block_size;
  int need = 0;
  for (int base = 0; base < p.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    const bool in = i < p.n;
    const int parent = in ? p.parents[i] : 0, child = in ? p.children[i] : 0, len = in ? p.lens[i] : 0;
    const int room = in && p.capacities ? p.capacities[i] : 0;
    unsigned int bad = 0;
    if (child < 0 || child >= p.t.rows || (len > 0 && (parent < 0 || parent >= p.t.rows))) bad |= kErrSeqId;
    if (len < 0 || room < 0) bad |= kErrInvalidRows;
    const int shared = max(len, 0) / bs;
    const int total = (int)(((long long)max(max(len, room), 0) + bs - 1) / bs);
    if (total > p.t.width) bad |= kErrTooManyBlocks;
    const int part = max(len, 0) - shared * bs;
    int from = kNoBlock, count = 1;  // the partial tokens' block, its count
    if (in && !bad) {
      // Both rows as they were before the round's claims.  (A claim of an earlier round is negative: its row is
      // neither empty nor long enough for a parent, as it would be refused within one round.)
      const int held = __ldcg(&p.t.seq_blocks[child]), of_parent = len > 0 ? __ldcg(&p.t.seq_blocks[parent]) : 0;
      if (part > 0) from = p.t.table[(long long)parent * p.t.width + shared];  // (shared < total <= width)
      if (held != 0 || (len > 0 && ((long long)len + bs - 1) / bs > of_parent)) bad |= kErrInvalidRows;
    }
    if (from < 0 || from >= p.c.num_blocks) from = kNoBlock;
    else count = p.t.refs[from];
    __syncthreads();
    // A row listed twice goes to its first child: the lowest claim wins.
    if (in && !bad) atomicMin(&p.t.seq_blocks[child], i - p.n);
    __syncthreads();
    if (in && !bad && __ldcg(&p.t.seq_blocks[child]) != i - p.n) bad |= kErrInvalidRows;
    if (in && bad) report(p.error_bits, bad);
    int all;
    const int before = block_scan(in && !bad ? total - shared : 0, sums, all);
    last = make_int4(shared, bad ? -1 : total, need + before, part);
    if (in) {
      reinterpret_cast<int4*>(p.plan)[i] = last;
      p.partial[i] = count > 0 ? from : kNoCount;
    }
    need += all;
  }
  return need;
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const __grid_constant__ ForkParams p) {
  extern __shared__ __align__(16) unsigned char plan_raw[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(plan_raw);
  pdl_trigger();
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  // The first CTA takes the children, the others the free blocks.
  const bool first = blockIdx.x == 0;
  PlanPart part{0, 0, 0};
  int is_free = 0, need = 0;
  int4 last = make_int4(0, -1, 0, 0);
  if (first) {
    need = plan_children(p, sh.sums, last);
  } else {
    part = plan_part(p.c.num_blocks, blockIdx.x - 1, kMapCtas);
    is_free = build_map(
        sh, part, p.t.refs, [](int r) { return r == 0; },
        [&](int at, bool in, int r) {
          const unsigned int word = __ballot_sync(~0u, in && r <= 0);
          if ((threadIdx.x & 31) == 0) p.uncounted[part.first / 32 + at] = word;
        });
  }
  asm volatile("barrier.cluster.wait;" ::: "memory");  // every CTA has started
  cluster_share(sh.cta_bits, is_free);
  cluster_share(sh.cta_more, need);
  cluster_sync();
  const int wanted = sh.cta_more[0];
  int before = 0, found = 0;
  for (int i = 0; i < kPlanCtas; ++i) {
    before += i < (int)blockIdx.x ? sh.cta_bits[i] : 0;
    found += sh.cta_bits[i];
  }
  if (!first && before < wanted)
    each_bit(sh, part.words, [&](int i, int rank) {
      if (before + rank < wanted) p.slots[before + rank] = (int)(part.first + i);
    });
  if (first) {
    for (int i = threadIdx.x; i < p.n; i += kPlanThreads) {
      const int4 plan = p.n <= kPlanThreads ? last : reinterpret_cast<const int4*>(p.plan)[i];
      if (plan.y < 0) continue;
      const int mine = plan.y - plan.x;
      const bool granted = mine == 0 || plan.z + mine <= found;
      if (!granted) {
        report(p.error_bits, kErrNoFreeBlock);
        p.plan[4 * i + 1] = -1;
      }
      p.t.seq_blocks[p.children[i]] = granted ? plan.y : 0;
    }
  }
}

constexpr int kEntries = 128;  // table entries that a warp takes at a time

__global__ void __launch_bounds__(kCopyThreads, kPartCtas) fork_kernel(const __grid_constant__ ForkParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  // The children's rows.
  const int per_row = (p.t.width + kEntries - 1) / kEntries;
  const long long warps = (long long)gridDim.x * kCopyWarps;
  for (long long unit = (long long)blockIdx.x * kCopyWarps + (threadIdx.x >> 5); unit < (long long)p.n * per_row;
       unit += warps) {
    const int i = (int)(unit / per_row), j0 = (int)(unit - (long long)i * per_row) * kEntries;
    const int4 plan = reinterpret_cast<const int4*>(p.plan)[i];
    const int shared = plan.x, total = plan.y;
    if (j0 >= total) continue;
    const int32_t* from = p.t.table + (long long)p.parents[i] * p.t.width;
    int32_t* to = p.t.table + (long long)p.children[i] * p.t.width;
    const int32_t* fresh = p.slots + plan.z - shared;
    int b[kEntries / 32];
#pragma unroll
    for (int u = 0; u < kEntries / 32; ++u) {
      const int j = j0 + lane + 32 * u;
      b[u] = j < shared ? from[j] : j < total ? fresh[j] : -1;
    }
    // Whether a shared block had a count is looked up as it was before the call: in a broken pool it may be one of
    // the fresh blocks too, and its count then rises by one for each row in either order.
    unsigned int lack[kEntries / 32];
#pragma unroll
    for (int u = 0; u < kEntries / 32; ++u)
      lack[u] = j0 + lane + 32 * u < shared && b[u] >= 0 && b[u] < p.c.num_blocks ? p.uncounted[b[u] >> 5] : 0u;
#pragma unroll
    for (int u = 0; u < kEntries / 32; ++u) {
      const int j = j0 + lane + 32 * u;
      if (j >= total) break;
      if (b[u] < 0 || b[u] >= p.c.num_blocks) {  // (of a shared one)
        report(p.error_bits, kErrBlockIndex);
        b[u] = -1;
      } else {
        atomicAdd(&p.t.refs[b[u]], 1);
        if ((lack[u] >> (b[u] & 31)) & 1) report(p.error_bits, kErrRefCount);
      }
      to[j] = b[u];
    }
  }
  // The partial blocks.  A pair takes two loads that depend on each other: once per CTA for the first children.
  auto look_up = [&](int i) {
    const int4 plan = reinterpret_cast<const int4*>(p.plan)[i];
    if (plan.y < 0 || plan.w == 0) return Pair{-1, -1, 0};
    return Pair{p.partial[i], p.slots[plan.z], plan.w};
  };
  __shared__ Pair known[kCopyThreads];
  if ((int)threadIdx.x < p.n) known[threadIdx.x] = look_up(threadIdx.x);
  __syncthreads();
  copy_pairs<kPartTiles>(
      p.c, p.n, [&](int i) { return i < kCopyThreads ? known[i] : look_up(i); },
      [&](int, const Pair& a) {
        if (a.tokens == 0) return false;
        if (a.src >= 0) return true;
        if (threadIdx.x == 0) report(p.error_bits, a.src == kNoCount ? kErrRefCount : kErrBlockIndex);
        return false;
      });
}

// ------------------------------------------------------------------------ free
struct FreeParams {
  Tables t;
  long long num_blocks;
  const int32_t* list;
  int n;
  unsigned int* error_bits;
};

// A CTA per row.  The first entries are loaded before the row's count is known.
__global__ void __launch_bounds__(1024) free_kernel(const __grid_constant__ FreeParams p) {
  __shared__ int held;
  constexpr int kAhead = 4;
  for (int i = blockIdx.x; i < p.n; i += gridDim.x) {
    const int row = p.list[i];
    if (row < 0 || row >= p.t.rows) {
      if (threadIdx.x == 0) report(p.error_bits, kErrSeqId);
      continue;
    }
    int32_t* entry = p.t.table + (long long)row * p.t.width;
    int ahead[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = threadIdx.x + u * blockDim.x;
      ahead[u] = j < p.t.width ? entry[j] : -1;
    }
    // Whoever takes the count frees the row: one that is listed twice is freed once.  (If it is, the entries
    // above may be another CTA's -1 by now; then the count is 0 and they are not used.)
    if (threadIdx.x == 0) {
      int n = atomicExch(&p.t.seq_blocks[row], 0);
      if (n < 0 || n > p.t.width) {
        report(p.error_bits, kErrTooManyBlocks);
        n = n < 0 ? 0 : p.t.width;
      }
      held = n;
    }
    __syncthreads();
    const int n = held;
    auto drop = [&](int j, int b) {
      entry[j] = -1;
      if (b < 0 || b >= p.num_blocks) {
        report(p.error_bits, kErrBlockIndex);
      } else if (atomicSub(&p.t.refs[b], 1) <= 0) {
        atomicAdd(&p.t.refs[b], 1);  // it was free already: a count never stays below what it was
        report(p.error_bits, kErrRefCount);
      }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = threadIdx.x + u * blockDim.x;
      if (j < n) drop(j, ahead[u]);
    }
    for (int j = threadIdx.x + kAhead * blockDim.x; j < n; j += blockDim.x) drop(j, entry[j]);
    __syncthreads();
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
};

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const __grid_constant__ CompactParams p) {
  extern __shared__ __align__(16) unsigned char plan_raw[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(plan_raw);
  pdl_trigger();
  const PlanPart part = plan_part(p.c.num_blocks, blockIdx.x, kPlanCtas);
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const int used = build_map(sh, part, p.t.refs, [](int r) { return r > 0; }, [](int, bool, int) {});
  asm volatile("barrier.cluster.wait;" ::: "memory");  // every CTA has started
  cluster_share(sh.cta_bits, used);
  cluster_sync();
  int live = 0, before = 0;  // blocks in use; those in earlier parts
  for (int i = 0; i < kPlanCtas; ++i) {
    before += i < (int)blockIdx.x ? sh.cta_bits[i] : 0;
    live += sh.cta_bits[i];
  }
  // Blocks in use below index `live` stay.  Block `live` lies in one part, which knows how many those are.
  const int low = (int)max(0ll, min((long long)part.count, live - part.first));  // the part's blocks below it
  int stay = 0;
  for (int w = threadIdx.x; w < part.words; w += kPlanThreads) {
    const int bits = low - 32 * w;
    stay += __popc(bits >= 32 ? sh.map[w] : bits > 0 ? sh.map[w] & ((1u << bits) - 1) : 0u);
  }
  int stay_part;
  block_scan(stay, sh.sums, stay_part);
  cluster_share(sh.cta_more, stay_part);
  cluster_sync();
  int stays = 0;
  for (int i = 0; i < kPlanCtas; ++i) stays += sh.cta_more[i];
  // The i-th free block below `live` takes the i-th block in use at or above it.
  const int lane = threadIdx.x & 31;
  int done = 0;
  for (int base = 0; base < part.words; base += kPlanThreads) {
    const int w0 = base + (int)(threadIdx.x & ~31);
    const unsigned int word = w0 + lane < part.words ? sh.map[w0 + lane] : 0u;
    int all;
    const int mine = done + before + block_scan(__popc(word), sh.sums, all);  // in use before the word's blocks
    done += all;
    for (int q = 0; q < 32 && w0 + q < part.words; ++q) {  // a word per step, a block per lane
      const unsigned int bits = __shfl_sync(~0u, word, q);
      const int in_use = __shfl_sync(~0u, mine, q) + __popc(bits & ((1u << lane) - 1));
      const int i = 32 * (w0 + q) + lane;
      const long long b = part.first + i;
      if (i >= part.count) continue;
      const bool is_used = (bits >> lane) & 1;
      p.new_index[b] = is_used ? (int)b : -1;  // (moved blocks get theirs below)
      if (b < live) {
        if (!is_used) p.dst[b - in_use] = (int)b;
      } else if (is_used) {
        p.src[in_use - stays] = (int)b;
      }
    }
  }
  const int moves = live - stays;
  if (blockIdx.x == 0 && threadIdx.x == 0) p.header[0] = moves;
  cluster_sync();
  for (int i = blockIdx.x * kPlanThreads + threadIdx.x; i < moves; i += kPlanCtas * kPlanThreads)
    p.new_index[__ldcg(p.src + i)] = __ldcg(p.dst + i);
}

__global__ void __launch_bounds__(kCopyThreads, kWholeCtas) compact_kernel(const __grid_constant__ CompactParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  // Table entries follow their blocks.
  const int per_row = (p.t.width + kEntries - 1) / kEntries;
  const long long warps = (long long)gridDim.x * kCopyWarps;
  for (long long unit = (long long)blockIdx.x * kCopyWarps + (threadIdx.x >> 5); unit < (long long)p.t.rows * per_row;
       unit += warps) {
    const int row = (int)(unit / per_row), j0 = (int)(unit - (long long)row * per_row) * kEntries;
    const int held = min(p.t.seq_blocks[row], p.t.width);
    if (j0 >= held) continue;
    int32_t* entry = p.t.table + (long long)row * p.t.width + j0;
    int b[kEntries / 32];
#pragma unroll
    for (int u = 0; u < kEntries / 32; ++u) b[u] = j0 + lane + 32 * u < held ? entry[lane + 32 * u] : -1;
#pragma unroll
    for (int u = 0; u < kEntries / 32; ++u) {
      if (j0 + lane + 32 * u >= held) break;
      if (b[u] < 0 || b[u] >= p.c.num_blocks) {
        report(p.error_bits, kErrBlockIndex);
        continue;
      }
      const int to = p.new_index[b[u]];
      if (to < 0) report(p.error_bits, kErrRefCount);
      if (to != b[u]) entry[lane + 32 * u] = to;
    }
  }
  // Blocks and counts.
  const int moves = p.header[0];
  for (int i = blockIdx.x * kCopyThreads + threadIdx.x; i < moves; i += gridDim.x * kCopyThreads) {
    p.t.refs[p.dst[i]] = p.t.refs[p.src[i]];
    p.t.refs[p.src[i]] = 0;
  }
  copy_pairs<kMoveTiles>(
      p.c, moves, [&](int i) { return Pair{p.src[i], p.dst[i], p.c.block_size}; },
      [](int, const Pair&) { return true; });
}

// ------------------------------------------------------------------------ host
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

// CTAs for a launch that copies up to `pairs` blocks and has `others` warps of other work.
static int copy_grid(const Caches& c, int ctas_per_sm, int tiles, long long pairs, long long others, unsigned& grid) {
  int dev = 0;
  NEB_CUDA(cudaGetDevice(&dev));
  const long long most = (long long)ctas_per_sm * num_sms(dev);
  NEB_REQUIRE(most > 0, NEB_ERR_CUDA, "could not size the grid for device %d", dev);
  const long long items = 2 * pairs * ((c.tiles + tiles - 1) / tiles), rest = (others + kCopyWarps - 1) / kCopyWarps;
  const long long ctas = items > rest ? items : rest;
  grid = (unsigned)(ctas < 1 ? 1 : ctas < most ? ctas : most);
  return NEB_OK;
}

static int check_plan_size(int64_t num_blocks) {
  NEB_REQUIRE(num_blocks <= kMaxPoolBlocks, NEB_ERR_UNSUPPORTED, "pools of more than %lld blocks are not supported",
              kMaxPoolBlocks);
  return NEB_OK;
}

// A plan kernel as one cluster.
template <typename P>
static int launch_plan(void (*kernel)(const P), const P& p, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  NEB_CUDA(cudaGetDevice(&dev));
  const size_t smem = plan_smem(p.c.num_blocks, kMapCtas);
  if (dev >= 64 || !ready[dev]) {
    NEB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)plan_smem(kMaxPoolBlocks, kMapCtas)));
    if (dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kPlanCtas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPlanCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  NEB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
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
  unsigned grid = 1;
  if (int rc = copy_grid(p.c, num_tokens ? kPartCtas : kWholeCtas, num_tokens ? kPartTiles : kWholeTiles, num_pairs,
                         0, grid)) return rc;
  (num_tokens ? copy_kernel<kPartCtas, kPartTiles> : copy_kernel<kWholeCtas, kWholeTiles>)<<<grid, kCopyThreads, 0,
                                                                   static_cast<cudaStream_t>(stream)>>>(p);
  NEB_CUDA(cudaGetLastError());
  return NEB_OK;
}

size_t neb_fork_workspace_bytes(int64_t num_blocks, int32_t num_children) {
  if (num_blocks <= 0 || num_blocks > INT_MAX || num_children < 0) return 0;
  return 20 * (size_t)num_children + 4 * (size_t)num_blocks + 4 * (((size_t)num_blocks + 31) / 32);
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
  if (int rc = check_plan_size(num_blocks)) return rc;
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
  p.partial = p.plan + 4ll * num_children;
  p.slots = p.partial + num_children;
  p.uncounted = reinterpret_cast<unsigned int*>(p.slots + num_blocks);
  p.error_bits = error_bits;
  unsigned grid = 1;
  const long long rows = (long long)num_children * (p.t.width / kEntries + 1);
  if (int rc = copy_grid(p.c, kPartCtas, kPartTiles, num_children, rows, grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = launch_plan(fork_plan_kernel, p, s)) return rc;
  NEB_CUDA(launch_pdl(fork_kernel, dim3(grid), dim3(kCopyThreads), 0, s, p));
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
  // As many threads as one round over a row can use.
  const int threads = max_blocks_per_seq <= 256 ? 256 : max_blocks_per_seq <= 512 ? 512 : 1024;
  free_kernel<<<num_rows, threads, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
  if (int rc = check_plan_size(num_blocks)) return rc;
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
  unsigned grid = 1;
  const long long rows = (long long)p.t.rows * (p.t.width / kEntries + 1);
  if (int rc = copy_grid(p.c, kWholeCtas, kMoveTiles, num_blocks / 2, rows, grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = launch_plan(compact_plan_kernel, p, s)) return rc;
  NEB_CUDA(launch_pdl(compact_kernel, dim3(grid), dim3(kCopyThreads), 0, s, p));
  return NEB_OK;
}

}  // extern "C"
