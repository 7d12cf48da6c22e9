// Log probabilities of logits rows: given token, rank, entropy, top alternatives.
//
// For a row x of V logits, M = max x and r = sum_j exp(x_j - M) without one element equal to M:
//   log p_j = (x_j - M) - log1p(r)
//   rank of t = 1 + #{j : x_j > x_t}
//   entropy = -sum_j p_j log p_j = log1p(r) - w / (1 + r),  w = sum_j exp(x_j - M) (x_j - M)
// so one pass over the row gives everything.  A running (m, s, w) takes a new
// maximum m' by s' = f s, w' = f (w + s (m - m')), f = exp(m - m'), and partial
// results join the same way.  Exponents are base 2 internally (t = (x - m) log2 e,
// ex2.approx), sums fp32.  r is kept apart from the maximum's own 1 because a
// confident row has log p = -log1p(r) with r << 1, which 1 + r would round away.
//
// A row is streamed by a cluster of S CTAs (S = 1 when the rows alone fill the
// GPU), each through a ring of 16 KB tiles filled by bulk asynchronous copies
// while the tiles before are summed from registers: the row is read once, the
// ring keeps the loads in flight whatever the arithmetic does.  The CTAs leave
// their sums and candidates in the first CTA's shared memory, so there is no
// workspace and no second launch.
//
// Alternatives: a CTA keeps a list of candidates and a threshold that at least
// num_top logits reach.  A tile's threads compare their own tile maximum (needed
// for m anyway) with the threshold, and only a thread above it looks at its
// logits again, so after the first tile almost no tile costs more than the
// barrier it needs to free its ring slot.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "neb_common.cuh"
#include "sm100.cuh"

namespace neb {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kWords = 4;                          // 16-byte words per thread and tile
constexpr int kTileWords = kThreads * kWords;      // 16 KB
constexpr int kStages = 3;
constexpr int kMaxTop = NEB_MAX_TOP_LOGPROBS;
constexpr int kMaxSplits = 8;                      // CTAs per row (the portable cluster size)
constexpr int kKeep = 64;                          // candidates left by a prune (at most)
constexpr int kList = kKeep + kMaxTop * kWords * 8;  // plus every logit of kMaxTop threads' tile
constexpr int kPruneAt = 192;                      // candidates from which a prune pays
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr long long kWaitLimit = 4000000000ll;     // cycles (about 2 s)

typedef unsigned long long u64;

struct Params {
  const void* logits;
  long long row_stride;
  int vocab, num_rows, num_top, splits;
  const int32_t* token_ids;
  float* logprobs;
  int32_t* ranks;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  unsigned int* error_bits;
};

// One CTA's part of a row: its maximum, the sums about it (r without the maximum itself).
struct Part {
  float m, r, w;
  int above;
};

struct Shared {
  uint4 ring[kStages][kTileWords];
  u64 list[kList];
  u64 sorted[kMaxTop];
  Part parts[kMaxSplits];
  u64 gathered[kMaxSplits][kMaxTop];
  uint64_t full[kStages];
  u64 warp_key[kWarps];
  float warp_f[3][kWarps];
  int warp_count[2][kWarps], warp_above[kWarps];
  int n, owner;
};

// ------------------------------------------------------------------- elements
template <typename T>
struct Elem;

// An unsigned order of fp32 values: NaN highest, -0 == +0.
__device__ __forceinline__ unsigned int order_f32(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned int b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of_order(unsigned int o) {
  if (o == 0xffffffffu) return __int_as_float(0x7fffffff);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ u64 make_key(float x, int idx) {
  return ((u64)order_f32(x) << 32) | (unsigned int)~(unsigned int)idx;
}
__device__ __forceinline__ int key_index(u64 key) { return (int)~(unsigned int)key; }
__device__ __forceinline__ float key_value(u64 key) { return value_of_order((unsigned int)(key >> 32)); }

template <>
struct Elem<__half> {
  static constexpr int kPerWord = 8;
  static constexpr unsigned int kLowest = 0xfc00fc00u;  // -inf pair
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __half2float(static_cast<const __half*>(p)[i]);
  }
  static __device__ __forceinline__ float2 pair(unsigned int u) { return h2_to_f2(u); }
  static __device__ __forceinline__ float get(const uint4& v, int j) {
    const unsigned int u = j < 4 ? (j < 2 ? v.x : v.y) : (j < 6 ? v.z : v.w);
    return __half2float(__ushort_as_half((unsigned short)((j & 1) ? u >> 16 : u)));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kPerWord = 8;
  static constexpr unsigned int kLowest = 0xff80ff80u;
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
  static __device__ __forceinline__ float2 pair(unsigned int u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ float get(const uint4& v, int j) {
    const unsigned int u = j < 4 ? (j < 2 ? v.x : v.y) : (j < 6 ? v.z : v.w);
    return __uint_as_float((j & 1) ? u & 0xffff0000u : u << 16);
  }
};
template <>
struct Elem<float> {
  static constexpr int kPerWord = 4;
  static constexpr unsigned int kLowest = 0xff800000u;
  static __device__ __forceinline__ float load(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ float get(const uint4& v, int j) {
    return __uint_as_float(j < 2 ? (j == 0 ? v.x : v.y) : (j == 2 ? v.z : v.w));
  }
};

// The two elements (of a pair word for 16-bit types, of two words for fp32) at position j of a word.
template <typename T>
__device__ __forceinline__ float2 word_pair(const uint4& v, int j) {
  if constexpr (Elem<T>::kPerWord == 8) {
    return Elem<T>::pair(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  } else {
    return j == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
}
template <typename T>
__device__ __forceinline__ float words_max(const uint4 (&v)[kWords]) {
  if constexpr (Elem<T>::kPerWord == 4) {
    float m = __int_as_float(0xff800000);
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[u].x), __uint_as_float(v[u].y)),
                         fmaxf(__uint_as_float(v[u].z), __uint_as_float(v[u].w))));
    }
    return m;
  } else if constexpr (sizeof(T) == 2 && Elem<T>::kLowest == 0xfc00fc00u) {
    __half2 m = __halves2half2(__ushort_as_half(0xfc00u), __ushort_as_half(0xfc00u));
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const unsigned int q[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2(m, *reinterpret_cast<const __half2*>(&q[i]));
    }
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    const unsigned int low = 0xff80ff80u;
    __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&low);
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const unsigned int q[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&q[i]));
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// Keeps a NaN, unlike fmaxf: a NaN logit has to reach the sums.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two fp32 lanes per instruction (sm_100).
__device__ __forceinline__ u64 pack2(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(u64 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// (from - to) log2 e for moving a reference up, finite also from an empty part (-inf).
__device__ __forceinline__ float step_down(float from, float to) { return fmaxf((from - to) * kLog2e, -1000.f); }

// Untiled bulk copy into shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   sm100::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
}

// ------------------------------------------------------------ block reductions
__device__ __forceinline__ int block_count(Shared& sh, int local, int& turn) {
  const int w = __reduce_add_sync(~0u, local);
  if ((threadIdx.x & 31) == 0) sh.warp_count[turn][threadIdx.x >> 5] = w;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) n += sh.warp_count[turn][i];
  turn ^= 1;
  return n;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The largest threshold search: a key `lo` with lowest <= #(keys > lo) <= most among the block's keys
// (mine(i) for i < mine_n, at least `lowest` of them above `lo` on entry).  Keys differ, so it exists.
template <typename F>
__device__ __forceinline__ u64 search(Shared& sh, int& turn, u64 lo, int lowest, int most, int mine_n, F mine) {
  u64 top = 0;
  for (int i = 0; i < mine_n; ++i) top = mine(i) > top ? mine(i) : top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(~0u, top, o);
    top = x > top ? x : top;
  }
  if ((threadIdx.x & 31) == 0) sh.warp_key[threadIdx.x >> 5] = top;
  __syncthreads();
  u64 hi = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) hi = sh.warp_key[i] > hi ? sh.warp_key[i] : hi;
  while (hi - lo > 1) {  // #(> lo) > most, #(> hi) < lowest
    const u64 mid = lo + (hi - lo) / 2;
    int c = 0;
    for (int i = 0; i < mine_n; ++i) c += mine(i) > mid;
    c = block_count(sh, c, turn);
    if (c >= lowest && c <= most) return mid;
    if (c > most) lo = mid; else hi = mid;
  }
  return lo;
}

// Leaves between num_top and kKeep of the list's n > kKeep candidates; returns the new threshold.
__device__ __noinline__ u64 prune(Shared& sh, int n, int num_top, int& turn) {
  constexpr int kEach = (kList + kThreads - 1) / kThreads;
  u64 key[kEach];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = threadIdx.x + i * kThreads;
    key[i] = at < n ? sh.list[at] : 0;
  }
  mine = kEach;
  const u64 thr = search(sh, turn, 0, num_top, kKeep, mine, [&](int i) { return key[i]; });
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (key[i] > thr) sh.list[atomicAdd(&sh.n, 1)] = key[i];
  __syncthreads();
  return thr;
}

// The list's num_top largest keys, in order, into sh.sorted (0 where there are fewer).
__device__ __forceinline__ void sort_top(Shared& sh, int n, int num_top, int& turn) {
  if (n > kKeep) {
    prune(sh, n, num_top, turn);
    n = sh.n;
  }
  if (threadIdx.x < num_top) sh.sorted[threadIdx.x] = 0;
  __syncthreads();
  if ((int)threadIdx.x < n) {
    const u64 key = sh.list[threadIdx.x];
    int before = 0;
    for (int j = 0; j < n; ++j) before += sh.list[j] > key;
    if (before < num_top) sh.sorted[before] = key;
  }
  __syncthreads();
}

// Joins `b` into `a`: sums about the larger maximum, which alone is left out of r.
__device__ __forceinline__ Part join(Part a, Part b) {
  if (b.m > a.m) {
    const Part t = a;
    a = b;
    b = t;
  }
  const float dt = step_down(b.m, a.m), f = fast_exp2(dt);
  const float s = b.m == neg_inf() ? b.r : 1.f + b.r;  // b's maximum is an ordinary term now
  a.r += f * s;
  a.w += f * (b.w + s * dt);
  a.above += b.above;
  return a;
}

// A row with a NaN or +inf, by the first CTA alone: results NaN, order over all values (NaN highest).
template <typename T>
__device__ __noinline__ void unordered_row(Shared& sh, const Params& p, const void* x, int row, int tok) {
  const int tid = threadIdx.x;
  const float nan = __int_as_float(0x7fffffff);
  int turn = 0;
  int above = 0;
  if (tok >= 0) {
    const unsigned int given = order_f32(Elem<T>::load(x, tok));
    for (int j = tid; j < p.vocab; j += kThreads) above += order_f32(Elem<T>::load(x, j)) > given;
  }
  above = block_count(sh, above, turn);
  if (tid == 0) {
    if (p.logprobs) p.logprobs[row] = nan;
    if (p.ranks) p.ranks[row] = tok >= 0 ? 1 + above : 0;
    if (p.entropy) p.entropy[row] = nan;
  }
  u64 limit = ~0ull;
  for (int k = 0; k < p.num_top; ++k) {
    u64 best = 0;
    for (int j = tid; j < p.vocab; j += kThreads) {
      const u64 key = make_key(Elem<T>::load(x, j), j);
      if (key < limit && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 n = __shfl_xor_sync(~0u, best, o);
      best = n > best ? n : best;
    }
    __syncthreads();
    if ((tid & 31) == 0) sh.warp_key[tid >> 5] = best;
    __syncthreads();
    limit = 0;
    for (int i = 0; i < kWarps; ++i) limit = sh.warp_key[i] > limit ? sh.warp_key[i] : limit;
    if (tid == 0) {
      p.top_ids[(long long)row * p.num_top + k] = key_index(limit);
      p.top_logprobs[(long long)row * p.num_top + k] = nan;
    }
  }
}

// --------------------------------------------------------------------- kernel
template <typename T>
__global__ void __launch_bounds__(kThreads, 3) token_logprobs_kernel(const Params p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  constexpr int kPer = Elem<T>::kPerWord;
  const int tid = threadIdx.x;
  const int splits = p.splits, row = blockIdx.x / splits, part = blockIdx.x - row * splits;
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.row_stride;
  const int k = p.num_top;

  // [head logits][16-byte words][tail logits]
  const int head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int words = (p.vocab - head) / kPer;
  const int tail = p.vocab - head - words * kPer;
  const int w0 = (int)((long long)words * part / splits), w1 = (int)((long long)words * (part + 1) / splits);
  const int tiles = (w1 - w0 + kTileWords - 1) / kTileWords;
  const uint4* xw = reinterpret_cast<const uint4*>(x + head) + w0;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&sh.full[i], 1);
    sm100::fence_mbar_init();
    sh.n = 0;
  }
  auto fill = [&](int tile) {  // by one thread
    const int st = tile % kStages;
    const uint32_t bytes = 16u * min(kTileWords, w1 - w0 - tile * kTileWords);
    sm100::mbar_arrive_expect_tx(&sh.full[st], bytes);
    bulk_load(sh.ring[st], xw + (long long)tile * kTileWords, bytes, &sh.full[st]);
  };
  if (tid == 0)
    for (int i = 0; i < min(kStages, tiles); ++i) fill(i);
  if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");

  int tok = p.token_ids ? p.token_ids[row] : -1;
  if (tok < -1 || tok >= p.vocab) {
    if (tid == 0 && part == 0 && p.error_bits) atomicOr(p.error_bits, kErrTokenId);
    tok = -1;
  }
  const float given = tok >= 0 ? Elem<T>::load(x, tok) : __int_as_float(0x7f800000);
  __syncthreads();

  float m = neg_inf(), s = 0.f, w = 0.f;  // sums about m, without the tile that holds m:
  float p_ref = 0.f;                      // that tile's sum
  int ref_tile = -1;                      // (-1: a head or tail logit, alone)
  int above = 0;
  u64 thr = 0;                            // at least k logits of this CTA are above it (0: not known yet)
  int n = k && part == 0 ? head + tail : 0;  // candidates listed so far
  int turn = 0;
  if (part == 0 && tid < head + tail) {
    const int j = tid < head ? tid : head + words * kPer + (tid - head);
    const float v = Elem<T>::load(x, j);
    if (v > m) m = v;
    const float t = max_nan((v - (m == neg_inf() ? 0.f : m)) * kLog2e, -200.f);
    p_ref = fast_exp2(t);
    above = v > given;
    if (k) sh.list[atomicAdd(&sh.n, 1)] = make_key(v, j);
  }

  bool late = false;
  for (int i = 0; i < tiles; ++i) {
    const int st = i % kStages;
    const int nw = w1 - w0 - i * kTileWords;  // words from this tile on
    if (!sm100::mbar_wait(&sh.full[st], (i / kStages) & 1, kWaitLimit)) late = true;
    uint4 v[kWords];
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const int a = tid + u * kThreads;
      v[u] = a < nw ? sh.ring[st][a]
                    : make_uint4(Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest);
    }
    const float tm = words_max<T>(v);
    const float mn = fmaxf(m, tm);
    {
      const float mm = mn == neg_inf() ? 0.f : mn;
      const u64 neg_m = pack2(-mm, -mm), c2 = pack2(kLog2e, kLog2e);
      u64 s0 = 0, s1 = 0, q0 = 0, q1 = 0;
#pragma unroll
      for (int u = 0; u < kWords; ++u) {
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) {
          const float2 f = word_pair<T>(v[u], j);
          const float2 t = unpack2(mul2(add2(pack2(f.x, f.y), neg_m), c2));
          const float tx = max_nan(t.x, -200.f), ty = max_nan(t.y, -200.f);
          const u64 e = pack2(fast_exp2(tx), fast_exp2(ty));
          if (j & 1) {
            s1 = add2(s1, e);
            q1 = fma2(e, pack2(tx, ty), q1);
          } else {
            s0 = add2(s0, e);
            q0 = fma2(e, pack2(tx, ty), q0);
          }
        }
      }
      const float2 sp = unpack2(add2(s0, s1)), qp = unpack2(add2(q0, q1));
      const float ps = sp.x + sp.y, pw = qp.x + qp.y;
      if (tm > m) {
        const float dt = step_down(m, mn), f = fast_exp2(dt), all = s + p_ref;
        w = fmaf(f, fmaf(all, dt, w), pw);
        s = f * all;
        p_ref = ps;
        ref_tile = i;
        m = mn;
      } else {
        s += ps;
        w += pw;
      }
    }
    if (__any_sync(~0u, tm > given)) {
#pragma unroll
      for (int u = 0; u < kWords; ++u)
#pragma unroll
        for (int j = 0; j < kPer; ++j) above += Elem<T>::get(v[u], j) > given;
    }
    if (k == 0) {
      __syncthreads();
      if (tid == 0 && i + kStages < tiles) fill(i + kStages);
      continue;
    }
    // ---- candidates
    const int base = head + (w0 + i * kTileWords + tid) * kPer;  // index of the thread's first logit
    const bool some = tid < nw;
    bool cand = some && make_key(tm, base) > thr;
    const int c = __syncthreads_count(cand);
    if (tid == 0 && i + kStages < tiles) fill(i + kStages);
    if (c == 0) continue;
    const int n0 = n;
    auto push = [&]() {
      if (!cand) return;
#pragma unroll
      for (int u = 0; u < kWords; ++u) {
        if (tid + u * kThreads < nw) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const u64 key = make_key(Elem<T>::get(v[u], j), base + u * kThreads * kPer + j);
            if (key > thr) {
              const int at = atomicAdd(&sh.n, 1);
              if (at < kList) sh.list[at] = key;
            }
          }
        }
      }
    };
    if (thr == 0) {
      // No threshold yet: each warp's ceil(k / warps)-th largest thread maximum; the
      // lowest of them is reached by at least k threads' maxima.
      unsigned int o = some ? order_f32(tm) : 0u, best = 0;
      for (int j = 0; j < (k + kWarps - 1) / kWarps; ++j) {
        best = __reduce_max_sync(~0u, o);
        const unsigned int who = __ballot_sync(~0u, o == best);
        if ((tid & 31) == __ffs(who) - 1) o = 0;
      }
      if ((tid & 31) == 0) sh.warp_key[tid >> 5] = best;
      __syncthreads();
      u64 low = ~0ull;
#pragma unroll
      for (int j = 0; j < kWarps; ++j) low = sh.warp_key[j] < low ? sh.warp_key[j] : low;
      if (low) {
        thr = (low << 32) - 1;
        cand = some && make_key(tm, base) > thr;
      }
    }
    push();
    __syncthreads();
    n = sh.n;
    if (n > kList) {
      // More than the list holds (equal or rising logits): drop this tile's, lower the
      // list to kKeep, and take a threshold that at most kMaxTop threads reach.
      __syncthreads();
      if (tid == 0) sh.n = n0;
      __syncthreads();
      n = n0;
      if (n0 > kKeep) {
        const u64 t = prune(sh, n0, k, turn);
        thr = t > thr ? t : thr;
        n = sh.n;
      }
      u64 best = 0;  // the thread's largest key
      if (some) {
#pragma unroll
        for (int u = kWords - 1; u >= 0; --u)
#pragma unroll
          for (int j = kPer - 1; j >= 0; --j) {
            const u64 key = make_key(Elem<T>::get(v[u], j), base + u * kThreads * kPer + j);
            if (tid + u * kThreads < nw && key > best) best = key;
          }
      }
      int over = block_count(sh, best > thr, turn);
      if (over > kMaxTop) {
        thr = search(sh, turn, thr, k, kMaxTop, 1, [&](int) { return best; });
      }
      cand = best > thr;
      __syncthreads();
      push();
      __syncthreads();
      n = sh.n;
    }
    if (n > kPruneAt) {
      const u64 t = prune(sh, n, k, turn);
      thr = t > thr ? t : thr;
      n = sh.n;
    }
  }

  // ---- this CTA's sums about its maximum
  {
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    if ((tid & 31) == 0) sh.warp_f[0][tid >> 5] = M;
    if (tid == 0) sh.owner = kThreads;
    __syncthreads();
    M = sh.warp_f[0][0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) M = fmaxf(M, sh.warp_f[0][i]);
    if (m == M && M != neg_inf()) atomicMin(&sh.owner, tid);
    __syncthreads();
    if (sh.owner == tid) {
      // Sum the tile that holds the maximum again, without it.
      float rest = p_ref != p_ref ? p_ref : 0.f;
      if (ref_tile >= 0) {
        bool left_out = false;
        for (int u = 0; u < kWords; ++u) {
          const int a = ref_tile * kTileWords + tid + u * kThreads;
          if (a >= w1 - w0) break;
          const uint4 word = __ldg(xw + a);
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const float f = Elem<T>::get(word, j);
            if (!left_out && f == M) left_out = true;
            else rest += fast_exp2(max_nan((f - M) * kLog2e, -200.f));
          }
        }
      }
      p_ref = rest;
    }
    const float dt = step_down(m, M), f = fast_exp2(dt), all = s + p_ref;
    const float r = warp_sum(f * all), q = warp_sum(f * fmaf(all, dt, w));
    const int up = __reduce_add_sync(~0u, above);
    const bool gave_up = __any_sync(~0u, late);
    if ((tid & 31) == 0) {
      sh.warp_f[1][tid >> 5] = r;
      sh.warp_f[2][tid >> 5] = q;
      sh.warp_above[tid >> 5] = up;
      if (gave_up && p.error_bits) atomicOr(p.error_bits, kErrTimeout);
    }
    if (k) sort_top(sh, n, k, turn);  // (its barriers also order the sums)
    else __syncthreads();
    Part mine{M, 0.f, 0.f, 0};
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      mine.r += sh.warp_f[1][i];
      mine.w += sh.warp_f[2][i];
      mine.above += sh.warp_above[i];
    }
    if (splits == 1) {
      if (tid == 0) sh.parts[0] = mine;
    } else {
      // Into the first CTA's shared memory.
      asm volatile("barrier.cluster.wait;" ::: "memory");  // it has started
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(sm100::smem_u32(&sh.parts[part])));
      if (tid == 0)
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(__float_as_uint(mine.m)),
                     "r"(__float_as_uint(mine.r)), "r"(__float_as_uint(mine.w)), "r"(mine.above)
                     : "memory");
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(sm100::smem_u32(&sh.gathered[part][0])));
      if (tid < k)
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at + 8 * tid), "l"(sh.sorted[tid]) : "memory");
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      if (part != 0) return;
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      if (k) {
        if (tid == 0) sh.n = 0;
        __syncthreads();
        for (int i = tid; i < splits * k; i += kThreads) {
          const u64 key = sh.gathered[i / k][i % k];
          if (key) sh.list[atomicAdd(&sh.n, 1)] = key;
        }
        __syncthreads();
        sort_top(sh, sh.n, k, turn);
      }
    }
    __syncthreads();
  }

  // ---- the row
  Part a = sh.parts[0];
  for (int i = 1; i < splits; ++i) a = join(a, sh.parts[i]);
  if (a.r != a.r || a.w != a.w) {
    unordered_row<T>(sh, p, x, row, tok);
    return;
  }
  const float nan = __int_as_float(0x7fffffff);
  const float ln_s = a.m == neg_inf() ? nan : log1pf(a.r);
  if (tid == 0) {
    if (p.logprobs) p.logprobs[row] = tok >= 0 ? (given - a.m) - ln_s : nan;
    if (p.ranks) p.ranks[row] = tok >= 0 ? 1 + a.above : 0;
    if (p.entropy) p.entropy[row] = ln_s - kLn2 * (a.w / (1.f + a.r));
  }
  if (tid < k) {
    const u64 key = sh.sorted[tid];
    p.top_ids[(long long)row * k + tid] = key_index(key);
    p.top_logprobs[(long long)row * k + tid] = (key_value(key) - a.m) - ln_s;
  }
}

// CTAs per row: enough for the GPU's resident CTAs (three per SM) when the rows alone are not, as long as
// each still has a tile to read.
static int choose_splits(long long rows, int vocab, int item, int sms) {
  const long long tiles = ((long long)vocab * item + 16 * kTileWords - 1) / (16 * kTileWords);
  int s = 1;
  while (s < kMaxSplits && 2 * s <= tiles && rows * s * 2 <= 3ll * sms) s *= 2;
  return s;
}

template <typename T>
static int launch(const Params& p, cudaStream_t stream, int device) {
  auto kernel = token_logprobs_kernel<T>;
  static bool ready[64] = {};
  if (device < 0 || device >= 64 || !ready[device]) {
    NEB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
    if (device >= 0 && device < 64) ready[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.num_rows * p.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  NEB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return NEB_OK;
}

}  // namespace logprobs
}  // namespace neb

using namespace neb;

extern "C" int neb_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, int32_t vocab,
                                  int32_t num_rows, const int32_t* token_ids, int32_t num_top, float* logprobs,
                                  int32_t* ranks, float* entropy, int32_t* top_ids, float* top_logprobs,
                                  uint32_t* error_bits, void* stream) {
  NEB_REQUIRE(dtype == NEB_DTYPE_F16 || dtype == NEB_DTYPE_BF16 || dtype == NEB_DTYPE_F32, NEB_ERR_INVALID,
              "unknown logits dtype %d", dtype);
  NEB_REQUIRE(num_rows >= 0 && vocab > 0 && row_stride >= 0, NEB_ERR_INVALID, "invalid sizes");
  NEB_REQUIRE(num_top >= 0 && num_top <= vocab && num_top <= NEB_MAX_TOP_LOGPROBS, NEB_ERR_INVALID,
              "num_top %d outside [0, min(vocab, %d)]", num_top, NEB_MAX_TOP_LOGPROBS);
  if (num_rows == 0) return NEB_OK;
  NEB_REQUIRE(logits, NEB_ERR_INVALID, "logits are null");
  NEB_REQUIRE((token_ids != nullptr) == (logprobs != nullptr) && (token_ids != nullptr) == (ranks != nullptr),
              NEB_ERR_INVALID, "token_ids, logprobs and ranks go together");
  NEB_REQUIRE(num_top == 0 || (top_ids && top_logprobs), NEB_ERR_INVALID, "top outputs are null");
  const int item = dtype == NEB_DTYPE_F32 ? 4 : 2;
  NEB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % item == 0, NEB_ERR_INVALID, "logits are misaligned");
  int dev = 0;
  NEB_CUDA(cudaGetDevice(&dev));
  logprobs::Params p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.num_rows = num_rows;
  p.num_top = num_top;
  p.splits = logprobs::choose_splits(num_rows, vocab, item, num_sms(dev));
  p.token_ids = token_ids;
  p.logprobs = logprobs;
  p.ranks = ranks;
  p.entropy = entropy;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  p.error_bits = error_bits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NEB_DTYPE_F16) return logprobs::launch<__half>(p, s, dev);
  if (dtype == NEB_DTYPE_BF16) return logprobs::launch<__nv_bfloat16>(p, s, dev);
  return logprobs::launch<float>(p, s, dev);
}
