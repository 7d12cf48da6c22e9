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
// GPU), each warp through a 4 KB tile of shared memory that a bulk asynchronous
// copy fills while the tile before is summed from registers.  No warp waits for
// another, and the row is read once.  The CTAs leave their sums and candidates in
// the first CTA's shared memory, so there is no workspace and no second launch.
//
// Alternatives: a CTA keeps a list of candidates and a threshold that num_top of
// them reach.  A lane compares its tile maximum (needed for m anyway) with the
// threshold, and only where it is higher does the warp look at that lane's logits
// again, in the tile, and list those above it.  The warp that lists every 8th (16th,
// 32nd: by num_top) candidate raises the threshold.  So after the first tile a tile
// costs one comparison, now and then a candidate, and no barrier: 2,048 rows of
// 151,936 fp16 logits list about 22 each for 5 alternatives, 90 for 20.
//
// What bounds it (device times in a graph): for many rows no unit alone.  2,048 of
// them take 110 us without alternatives, 5.7 TB/s, 128 us with 5, 153 us with 20
// (reading them alone in this way 105 us; exp2, one per logit, is 69 us of the XU
// pipe); two full waves under the profiler keep HBM busy for 51 % of the time, the
// issue slots for 57 % and XU for 54 %.  The rest is latency at the start and the
// end of each row, which the other two CTAs of the SM hide in part.  For few rows
// it is latency alone: one row 6.8 us, with 20 alternatives 12 us, of which the
// launch, the first tile and the joins are all but 2 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "neb_common.cuh"
#include "sm100.cuh"

namespace neb {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kWords = 8;                  // 16-byte words per lane and tile
constexpr int kTileWords = 32 * kWords;    // of one warp: 4 KB
constexpr int kCtas = 3;                   // resident per SM
constexpr int kMaxTop = NEB_MAX_TOP_LOGPROBS;
constexpr int kMaxSplits = 8;              // CTAs per row (the portable cluster size)
constexpr int kList = 512;                 // candidates
constexpr int kWindow = 128;               // the last candidates, which a higher threshold is taken from
constexpr int kMaxVocab = 1 << 30;         // (an index in int with tiles to spare)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kWaitNs = 20000;        // of sleep between two looks at a tile
constexpr long long kWaitLimit = 4000000000ll;  // cycles (about 2 s)

typedef unsigned long long u64;

struct Params {
  const void* logits;
  long long row_stride;
  int vocab, num_rows, num_top, splits;  // splits: CTAs per row
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
  int above;  // logits larger than the given token's (bit 31: see kSkipped)
};
constexpr int kSkipped = INT_MIN;  // a tile below kLow was left out

struct Shared {
  uint4 slot[kWarps][kTileWords];
  u64 list[kList];
  u64 sorted[kMaxTop], merged[kMaxTop];  // the part's largest keys, the row's
  Part parts[kMaxSplits];
  u64 gathered[kMaxSplits * kMaxTop];  // num_top of each part
  uint64_t full[kWarps];
  u64 warp_key[kWarps];
  int first_index[kWarps];  // of each warp's range
  unsigned int tops[64];
  u64 threshold;  // only larger keys are listed; num_top listed ones are at or above it
  float warp_f[4][kWarps];
  int warp_count[2][kWarps], warp_above[kWarps];
  int n;  // candidates offered (beyond kList: not all are listed)
};

// ------------------------------------------------------------------- elements
// Keeps a NaN, unlike fmaxf.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

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

// The one-pass sums are for rows whose maximum lies in [kLowRow, kHighRow], where the rounding of m log2 e
// stays small and clamped differences finite; other rows go to general_row.  Logits below kLow (masks by a
// large negative number) are never a reference: beside such a maximum their share is exp(-1000) or less.
constexpr float kLow = -65000.f, kLowRow = -64000.f, kHighRow = 66000.f;
constexpr float kFinite = -65504.f;
// The threshold below every key but those of such masked logits.
__device__ __forceinline__ u64 no_masked() { return ((u64)order_f32(kLow) << 32) - 1; }

template <>
struct Elem<__half> {
  typedef __half2 Two;
  static constexpr int kPerWord = 8;
  static constexpr unsigned int kLowest = 0xfc00fc00u;  // -inf pair
  static constexpr float kUlp = 1.f / 512.f;  // of the type, relative
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __half2float(static_cast<const __half*>(p)[i]);
  }
  static __device__ __forceinline__ float2 pair(unsigned int u) { return h2_to_f2(u); }
  static __device__ __forceinline__ Two twice(float x) { return __float2half2_rn(x); }
};
template <>
struct Elem<__nv_bfloat16> {
  typedef __nv_bfloat162 Two;
  static constexpr int kPerWord = 8;
  static constexpr unsigned int kLowest = 0xff80ff80u;
  static constexpr float kUlp = 1.f / 64.f;  // of the type, relative
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
  static __device__ __forceinline__ float2 pair(unsigned int u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ Two twice(float x) { return __float2bfloat162_rn(x); }
};
template <>
struct Elem<float> {
  static constexpr int kPerWord = 4;
  static constexpr unsigned int kLowest = 0xff800000u;
  static constexpr float kUlp = 0.f;  // of the type, relative
  static __device__ __forceinline__ float load(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
};

// The 32-bit piece q of a word, and its one or two logits.
__device__ __forceinline__ unsigned int piece(const uint4& v, int q) {
  return q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
}
// NaN if there is one.
template <typename T, int N>
__device__ __forceinline__ float words_max(const uint4 (&v)[N]) {
  if constexpr (Elem<T>::kPerWord == 4) {
    float m = neg_inf();
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) m = max_nan(m, __uint_as_float(piece(v[u], q)));
    return m;
  } else {
    typedef typename Elem<T>::Two Two;
    const unsigned int low = Elem<T>::kLowest;
    Two m = *reinterpret_cast<const Two*>(&low);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned int x = piece(v[u], q);
        m = __hmax2_nan(m, *reinterpret_cast<const Two*>(&x));
      }
    return max_nan(__low2float(m), __high2float(m));
  }
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
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A step of the exponent's reference, finite also from an empty part (-inf).
__device__ __forceinline__ float bounded(float step) { return fmaxf(step, -1000.f); }

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The exponents' reference: t = x log2 e - mc with mc the rounded m log2 e, one fma per logit.  t of m
// itself is t0, not 0; e0 = 2^t0 takes that out of the finished sums.
__device__ __forceinline__ float exponent(float x, float mc) { return fmaf(x, kLog2e, -mc); }

// Moves the sums to the reference `top`.
__device__ __forceinline__ void move_up(float top, float& m, float& mc, float& s, float& w, float& p_ref) {
  const float to = top * kLog2e, dt = bounded(m == neg_inf() ? -1000.f : mc - to), f = fast_exp2(dt);
  const float all = s + p_ref;
  w = f * fmaf(all, dt, w);
  s = f * all;
  p_ref = 0.f;
  m = top;
  mc = to;
}

// Where logits far below the reference are cut off: their terms are 0 all the same.
template <typename T>
__device__ __forceinline__ float low_end(float m) {
  return fmaxf(m - 100.f - fabsf(m) * Elem<T>::kUlp, kFinite);
}

// Adds the words' terms 2^t and 2^t t, two fp32 lanes per instruction.  The cut-off keeps
// 0 times -inf out of the second sum.
template <typename T, int N>
__device__ __forceinline__ void add_words(const uint4 (&v)[N], float m, float mc, u64& s, u64& w) {
  const u64 c2 = pack2(kLog2e, kLog2e), mc2 = pack2(-mc, -mc);
  const float lo = low_end<T>(m);
  auto add = [&](float a, float b) {
    const u64 t = fma2(pack2(a, b), c2, mc2);
    const float2 f = unpack2(t);
    const u64 e = pack2(fast_exp2(f.x), fast_exp2(f.y));
    s = add2(s, e);
    w = fma2(e, t, w);
  };
  if constexpr (Elem<T>::kPerWord == 4) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      add(fmaxf(__uint_as_float(v[u].x), lo), fmaxf(__uint_as_float(v[u].y), lo));
      add(fmaxf(__uint_as_float(v[u].z), lo), fmaxf(__uint_as_float(v[u].w), lo));
    }
  } else {
    typedef typename Elem<T>::Two Two;
    const Two lo2 = Elem<T>::twice(lo);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned int x = piece(v[u], q);
        const Two h = __hmax2(*reinterpret_cast<const Two*>(&x), lo2);
        const float2 f = Elem<T>::pair(*reinterpret_cast<const unsigned int*>(&h));
        add(f.x, f.y);
      }
  }
}

// Logits larger than `given`.
template <typename T, int N>
__device__ __forceinline__ int count_above(const uint4 (&v)[N], float given) {
  if constexpr (Elem<T>::kPerWord == 4) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) n += __uint_as_float(piece(v[u], q)) > given;
    return n;
  } else {
    typedef typename Elem<T>::Two Two;
    const Two g = Elem<T>::twice(given);  // exact: it is one of the logits
    // Masks 0xffff add up to 65536 (low - high) - low in 32 bits.
    unsigned int sum = 0;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned int x = piece(v[u], q);
        sum += __hgt2_mask(*reinterpret_cast<const Two*>(&x), g);
      }
    const int low = (int)(-sum & 0xffffu);
    return 2 * low - ((int)(sum + low) >> 16);
  }
}

// Untiled bulk copy into shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   sm100::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
}

// The warp's wait for its tile: bounded, asleep between looks (the other warps need the issue slots).
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity) {
  bool ok = sm100::mbar_try_wait_sleep(bar, parity, kWaitNs);
  if (!ok) {
    const long long t0 = clock64();
    do {
      ok = sm100::mbar_try_wait_sleep(bar, parity, kWaitNs);
    } while (!ok && clock64() - t0 < kWaitLimit);
  }
  return __all_sync(~0u, ok);
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

// A key `lo` with lowest <= #(keys > lo) <= most among the block's keys (mine(i) for i < mine_n, more than `most`
// of them above `lo` on entry).  Keys differ, so it exists.
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

// The num_top largest of n keys in order into `sorted`, by counting; its places beyond n keep their 0.  Keys of
// 0 are none.
__device__ __forceinline__ void rank_keys(const u64* keys, int n, int num_top, u64* sorted) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const u64 key = keys[i];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += keys[j] > key;
    if (key && before < num_top) sorted[before] = key;
  }
  __syncthreads();
}

// Lists the logits above the threshold among the words of the warp's candidate lanes, a 32-bit piece of the
// tile per lane.  `from`: the tile's first word in the warp's range, `value` the threshold's.  True when it is time
// for a better threshold.
template <typename T>
__device__ __forceinline__ bool list_candidates(Shared& sh, int from, int words, bool cand, float value, int k) {
  constexpr int kPer = Elem<T>::kPerWord;
  static_assert(kWords * 4 == 32, "a lane's words are one piece per lane");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, word = (lane >> 2) * 32;
  const unsigned int* piece_of = reinterpret_cast<const unsigned int*>(sh.slot[warp] + word) + (lane & 3);
  const int first = sh.first_index[warp] + from * kPer;
  const int every = k <= 8 ? 8 : k <= 16 ? 16 : 32;
  const u64 thr = *static_cast<volatile u64*>(&sh.threshold);
  if (__any_sync(~0u, *static_cast<volatile int*>(&sh.n) > kList)) return false;  // (one answer for the warp)
  bool due = false;
  auto offer = [&](float f, int idx) {
    const u64 key = make_key(f, idx);
    if (key > thr) {
      const int to = atomicAdd(&sh.n, 1);
      if (to < kList) sh.list[to] = key;
      due |= ((to + 1) & (every - 1)) == 0;
    }
  };
  for (unsigned int left = __ballot_sync(~0u, cand); left; left &= left - 1) {
    const int other = __ffs(left) - 1;
    if (other + word < words) {
      const unsigned int x = piece_of[4 * other];
      const int at = first + (other + word) * kPer + (lane & 3) * (kPer / 4);
      if constexpr (kPer == 8) {
        const float2 f = Elem<T>::pair(x);
        if (fmaxf(f.x, f.y) >= value) {
          if (f.x >= value) offer(f.x, at);
          if (f.y >= value) offer(f.y, at + 1);
        }
      } else {
        if (__uint_as_float(x) >= value) offer(__uint_as_float(x), at);
      }
    }
  }
  return __any_sync(~0u, due);
}

// Raises the threshold to a value that num_top of the last candidates exceed, and few more: a search by halves,
// some eight steps, by one warp.  (Counting each candidate's place instead made 20 alternatives of 2,048 rows 45 us
// slower.)  Others may be listing meanwhile: a place that is not written yet holds 0, which only makes the
// threshold lower.
__device__ __noinline__ void raise_threshold(Shared& sh, int num_top) {
  const int lane = threadIdx.x & 31;
  // (What others may change is read by one lane: the votes below need one course for the warp.)
  const int n = min(__shfl_sync(~0u, *static_cast<volatile int*>(&sh.n), 0), kList), from = max(0, n - kWindow);
  unsigned int lo = __shfl_sync(~0u, reinterpret_cast<volatile unsigned int*>(&sh.threshold)[1], 0);
  unsigned int v[kWindow / 32], hi = 0, best = 0;
#pragma unroll
  for (int i = 0; i < kWindow / 32; ++i) {
    const int at = from + lane + 32 * i;
    v[i] = at < n ? reinterpret_cast<volatile unsigned int*>(&sh.list[at])[1] : 0u;
    hi = max(hi, v[i]);
  }
  hi = __reduce_max_sync(~0u, hi);
  for (int step = 0; step < 12 && hi > lo + 1; ++step) {  // fewer than num_top exceed `hi`
    const unsigned int mid = lo + (hi - lo) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kWindow / 32; ++i) c += __popc(__ballot_sync(~0u, v[i] > mid));
    if (c >= num_top) {
      best = lo = mid;
      if (c <= num_top + num_top / 4) break;
    } else {
      hi = mid;
    }
  }
  if (best && lane == 0) atomicMax(&sh.threshold, ((u64)best << 32) | 0xffffffffu);
}

// The num_top largest keys above `thr` of a row part whose list ran over (equal or rising logits) or of a whole row,
// word by word from memory: in order in sh.list.  Returns how many.
template <typename T>
__device__ __noinline__ int collect(Shared& sh, const uint4* data, int words, int first, const void* x, int vocab,
                                    int head, int tail, int k, u64 thr) {
  constexpr int kPer = Elem<T>::kPerWord;
  constexpr int kMost = kThreads - kMaxTop;
  const int tid = threadIdx.x;
  int turn = 0, n = 0;
  for (int base = 0; base == 0 || base < words; base += kThreads) {
    u64 key[kPer + 1] = {};
    if (base + tid < words) {
      for (int j = 0; j < kPer; ++j) {
        const long long at = (long long)(base + tid) * kPer + j;
        key[j] = make_key(Elem<T>::load(data, at), first + (int)at);
      }
    }
    if (base == 0 && tid < head + tail) {
      const int at = tid < head ? tid : vocab - tail + (tid - head);
      key[kPer] = make_key(Elem<T>::load(x, at), at);
    }
    int c = 0;
    for (int j = 0; j <= kPer; ++j) c += key[j] > thr;
    c = block_count(sh, c, turn);
    if (c == 0) continue;
    if (c > kMost) thr = search(sh, turn, thr, k, kMost, kPer + 1, [&](int j) { return key[j]; });
    if (tid == 0) sh.n = n;
    __syncthreads();
    for (int j = 0; j <= kPer; ++j)
      if (key[j] > thr) sh.list[atomicAdd(&sh.n, 1)] = key[j];
    __syncthreads();
    n = sh.n;
    if (tid < k) sh.sorted[tid] = 0;
    __syncthreads();
    rank_keys(sh.list, n, k, sh.sorted);
    n = min(n, k);
    if (tid < n) sh.list[tid] = sh.sorted[tid];
    if (n == k) thr = sh.sorted[k - 1] > thr ? sh.sorted[k - 1] : thr;
    __syncthreads();
  }
  return n;
}

// Fills `sorted` from n to k with the logits below kLow, which the candidates leave out: largest first (all of
// them mostly equal, -inf or another mask), then by index.  A pass over the row for the next lower value, four
// words per thread in flight, and its first logits: 5 allowed tokens of 151,936 with 20 alternatives take 19 us in
// place of 13 (one row, the others -inf).  It is made for few distinct masked values: where each differs (x - 1e5
// in fp32) there is a pass for every alternative that the allowed tokens do not fill, 3 ms for such a row.
template <typename T>
__device__ __noinline__ void fill_masked(Shared& sh, u64* sorted, const void* x, int vocab, int head, int n, int k) {
  constexpr int kPer = Elem<T>::kPerWord;
  const int tid = threadIdx.x, words = (vocab - head) / kPer;
  const uint4* data = reinterpret_cast<const uint4*>(static_cast<const T*>(x) + head);
  int turn = 0;
  float limit = kLow;
  while (n < k) {
    float next = neg_inf();
    bool any = false;
    auto look = [&](float v) {
      if (v < limit) {
        next = fmaxf(next, v);
        any = true;
      }
    };
    for (int base = tid; base < words; base += 4 * kThreads) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (base + u * kThreads < words) v[u] = __ldg(data + base + u * kThreads);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (base + u * kThreads >= words) break;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (kPer == 8) {
            const float2 f = Elem<T>::pair(piece(v[u], q));
            look(f.x);
            look(f.y);
          } else {
            look(__uint_as_float(piece(v[u], q)));
          }
        }
      }
    }
    for (int j = tid; j < vocab - words * kPer; j += kThreads) look(Elem<T>::load(x, j < head ? j : j + words * kPer));
    unsigned int best = any ? order_f32(next) : 0u;
    best = __reduce_max_sync(~0u, best);
    __syncthreads();
    if ((tid & 31) == 0) sh.warp_key[tid >> 5] = best;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) best = max(best, (unsigned int)sh.warp_key[i]);
    if (best == 0) break;  // (not reached: k is at most the vocabulary)
    for (int base = 0; base < vocab && n < k; base += kThreads) {
      const int j = base + tid;
      const bool hit = j < vocab && order_f32(Elem<T>::load(x, j)) == best;
      const unsigned int who = __ballot_sync(~0u, hit);
      if ((tid & 31) == 0) sh.warp_count[turn][tid >> 5] = __popc(who);
      __syncthreads();
      int before = __popc(who & ((1u << (tid & 31)) - 1)), all = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < (tid >> 5)) before += sh.warp_count[turn][i];
        all += sh.warp_count[turn][i];
      }
      turn ^= 1;
      if (hit && n + before < k) sorted[n + before] = ((u64)best << 32) | (unsigned int)~(unsigned int)j;
      n += all;
    }
    limit = value_of_order(best);
  }
  __syncthreads();
}

// A lane's terms of the tile at `data`, but for the logits equal to the maximum M, which it counts.  (All loads
// come before the first use, so that the warp waits once.)
template <typename T>
__device__ __noinline__ float tile_without(const uint4* data, int words, float M, float m, float mc, int& equal) {
  uint4 v[kWords];
#pragma unroll
  for (int u = 0; u < kWords; ++u) {
    const int a = (threadIdx.x & 31) + u * 32;
    v[u] = a < words ? __ldg(data + a)
                     : make_uint4(Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest);
  }
  const float lo = low_end<T>(m);
  float sum = 0.f;
  int n = 0;
  auto take = [&](float f) {
    const float e = fast_exp2(exponent(fmaxf(f, lo), mc));
    n += f == M;
    sum += f == M ? 0.f : e;
  };
#pragma unroll
  for (int u = 0; u < kWords; ++u) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (Elem<T>::kPerWord == 8) {
        const float2 f = Elem<T>::pair(piece(v[u], q));
        take(f.x);
        take(f.y);
      } else {
        take(__uint_as_float(piece(v[u], q)));
      }
    }
  }
  equal = n;
  return sum;
}

// Joins the parts, one per lane of each warp (kMaxSplits at most): sums about the row's maximum, which alone is
// left out of r.
__device__ __forceinline__ Part join(const Part* parts, int n) {
  const int lane = threadIdx.x & 31;
  Part a = parts[lane < n ? lane : 0];
  if (lane >= n) a = Part{neg_inf(), 0.f, 0.f, 0};
  const float M = warp_max_nan(a.m);
  const unsigned int top = __ballot_sync(~0u, a.m == M);
  const float dt = bounded((a.m - M) * kLog2e), f = fast_exp2(dt);
  const float own = a.m == neg_inf() || lane == __ffs(top) - 1 ? 0.f : 1.f;  // the part's maximum as an ordinary term
  Part r;
  r.m = M;
  r.r = warp_sum(f * (own + a.r));
  r.w = warp_sum(f * (a.w + (own + a.r) * dt));
  const unsigned int skipped = __reduce_or_sync(~0u, (unsigned int)a.above) & (unsigned int)kSkipped;
  r.above = __reduce_add_sync(~0u, a.above & INT_MAX) | (int)skipped;
  return r;
}

// Any row, logit by logit from memory, by one CTA: rows with a NaN or +inf (results NaN, order over all values),
// rows whose maximum lies outside [kLowRow, kHighRow], and rows that lost a tile.  Slow, as such rows are rare:
// 151,936 fp16 logits at the lowest value 42 us, with 20 alternatives 100 us (their largest in one pass of keys; a
// pass per alternative took 619 us), beside the 6 us and 12 us of another row (device times in a graph).
template <typename T>
__device__ __noinline__ void general_row(Shared& sh, const Params& p, const void* x, int row, int head, int tok) {
  const int tid = threadIdx.x;
  const float nan = __int_as_float(0x7fffffff);
  int turn = 0, above = 0;
  float m = neg_inf();
  const unsigned int given = tok >= 0 ? order_f32(Elem<T>::load(x, tok)) : ~0u;
  for (int j = tid; j < p.vocab; j += kThreads) {
    const float v = Elem<T>::load(x, j);
    above += order_f32(v) > given;
    m = fmaxf(m, v);
  }
  above = block_count(sh, above, turn);
  m = warp_max_nan(m);
  if ((tid & 31) == 0) sh.warp_f[0][tid >> 5] = m;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) m = fmaxf(m, sh.warp_f[0][i]);
  float s = 0.f, w = 0.f;
  for (int j = tid; j < p.vocab; j += kThreads) {
    const float t = (Elem<T>::load(x, j) - m) * kLog2e;  // NaN where the row's results are
    const float e = fast_exp2(t);
    s += e;
    if (!(e == 0.f)) w = fmaf(e, t, w);
  }
  s = warp_sum(s);
  w = warp_sum(w);
  if ((tid & 31) == 0) {
    sh.warp_f[1][tid >> 5] = s;
    sh.warp_f[2][tid >> 5] = w;
  }
  __syncthreads();
  s = w = 0.f;
  for (int i = 0; i < kWarps; ++i) {
    s += sh.warp_f[1][i];
    w += sh.warp_f[2][i];
  }
  float r = s - 1.f;
  if (s < 2.f) {  // a confident row: summed again without its maximum
    r = 0.f;
    for (int j = tid; j < p.vocab; j += kThreads) {
      const float v = Elem<T>::load(x, j);
      r += v == m ? 0.f : fast_exp2((v - m) * kLog2e);
    }
    r = warp_sum(r);
    if ((tid & 31) == 0) sh.warp_f[3][tid >> 5] = r;
    __syncthreads();
    r = 0.f;
    for (int i = 0; i < kWarps; ++i) r += sh.warp_f[3][i];
  }
  const float ln_s = log1pf(r);
  if (tid == 0) {
    if (p.logprobs) p.logprobs[row] = tok >= 0 ? (Elem<T>::load(x, tok) - m) - ln_s : nan;
    if (p.ranks) p.ranks[row] = tok >= 0 ? 1 + above : 0;
    if (p.entropy) p.entropy[row] = ln_s - kLn2 * (w / (1.f + r));
  }
  const int k = p.num_top;
  if (k == 0) return;
  constexpr int kPer = Elem<T>::kPerWord;
  const int words = (p.vocab - head) / kPer, tail = p.vocab - head - words * kPer;
  const uint4* data = reinterpret_cast<const uint4*>(static_cast<const T*>(x) + head);
  collect<T>(sh, data, words, head, x, p.vocab, head, tail, k, 0);  // (every key is above 0)
  if (tid < k) {
    const u64 key = sh.list[tid];
    p.top_ids[(long long)row * k + tid] = key_index(key);
    p.top_logprobs[(long long)row * k + tid] = (key_value(key) - m) - ln_s;
  }
}

// What the CTA reads: [head logits][16-byte words][tail logits] of its row, the words in parts, a part in a range
// for each warp.
template <typename T>
struct Place {
  const T* x;
  const uint4* data;  // the part's words
  int row, part, head, tail, w0, words, share;  // of the row; of the part; words of a warp
  __device__ __forceinline__ explicit Place(const Params& p) {
    row = blockIdx.x / (unsigned)p.splits;
    part = blockIdx.x - row * p.splits;
    x = static_cast<const T*>(p.logits) + (long long)row * p.row_stride;
    head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int all = (p.vocab - head) / Elem<T>::kPerWord;
    tail = p.vocab - head - all * Elem<T>::kPerWord;
    const int even = (unsigned)all / (unsigned)p.splits, more = all - even * p.splits;  // `more` parts have one more
    w0 = part * even + min(part, more);
    words = even + (part < more);
    data = reinterpret_cast<const uint4*>(x + head) + w0;
    share = ((words + kThreads - 1) / kThreads) * 32;
  }
  __device__ __forceinline__ int first_word() const { return (int)(threadIdx.x >> 5) * share; }
  __device__ __forceinline__ int mine() const { return min(share, words - first_word()); }  // (0 or less: none)
  __device__ __forceinline__ int index(int word) const { return head + (w0 + word) * Elem<T>::kPerWord; }
};

// --------------------------------------------------------------------- kernel
// The rest of a row part: head and tail logits, the sums of the warps and of the parts, the row's results.  Out of
// line, so that its registers are not the loop's.
template <typename T>
__device__ __noinline__ void finish(Shared& sh, const Params& p, float m, float mc, float s, float w, float p_ref,
                                    float given, int above, int ref_tile) {
  const Place<T> at(p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int splits = p.splits, row = at.row, part = at.part, head = at.head, tail = at.tail, k = p.num_top;
  float lone = neg_inf();  // a lane's head or tail logit
  if (part == 0 && warp == 0 && head + tail > 0) {
    const int index = lane < head ? lane : p.vocab - tail + (lane - head);
    if (lane < head + tail) lone = Elem<T>::load(at.x, index);
    const float top = warp_max_nan(lone);
    if (top > m && top >= kLow) {
      move_up(top, m, mc, s, w, p_ref);
      ref_tile = -1;
    }
    if (lone >= kLow) {
      const float t = exponent(fmaxf(lone, low_end<T>(m)), mc), e = fast_exp2(t);
      if (ref_tile < 0) p_ref = e;
      else s += e;
      w = fmaf(e, t, w);
    }
    if (top != top) s = top;
    else if (m == neg_inf() && top > neg_inf()) above |= kSkipped;
    above += lone > given;
    if (k) {
      const u64 key = make_key(lone, index);
      if (key > *static_cast<volatile u64*>(&sh.threshold)) {
        const int to = atomicAdd(&sh.n, 1);
        if (to < kList) sh.list[to] = key;
      }
    }
  }

  // ---- this CTA's sums about its maximum
  {
    if (lane == 0) sh.warp_f[0][warp] = m;
    __syncthreads();
    float M = sh.warp_f[0][0];
    int owner = 0;
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
      const float other = sh.warp_f[0][i];
      owner = other > M ? i : owner;
      M = fmaxf(M, other);
    }
    // The part's sum with its maximum, for a first look: from 2 on, subtracting the maximum's 1 loses nothing.
    const float dt = bounded((m - M) * kLog2e), f = fast_exp2(dt), t0 = m == neg_inf() ? 0.f : exponent(m, mc),
                inv = fast_exp2(-t0);
    {
      const float look = warp_sum(f * inv * (s + p_ref));
      if (lane == 0) sh.warp_f[1][warp] = look;
    }
    __syncthreads();
    float S = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) S += sh.warp_f[1][i];
    const bool apart = S < 2.f;
    if (apart && owner == warp && M != neg_inf()) {
      // Sum the tile that holds the maximum again, without it.
      float rest = p_ref != p_ref ? p_ref : 0.f;
      int equal = 0;  // logits equal to the maximum
      if (ref_tile < 0) {
        equal = lone == M;
        if (!equal && !(lone < kLow)) rest += fast_exp2(exponent(fmaxf(lone, low_end<T>(m)), mc));
      } else {
        rest += tile_without<T>(at.data + at.first_word() + ref_tile, at.mine() - ref_tile, M, m, mc, equal);
      }
      const unsigned int who = __ballot_sync(~0u, equal > 0);
      const float e0 = fast_exp2(exponent(m, mc));
      if (lane == __ffs(who) - 1) --equal;
      p_ref = fmaf((float)equal, e0, rest);
    }
    // From the rounded reference to m, then to the CTA's maximum.  The maximum itself, left out of the owner's
    // sum, has a term in w: e0 t0.
    const float all = s + p_ref, left_out = apart && owner == warp && lane == 0 ? fast_exp2(t0) : 0.f;
    const float q = (w - t0 * (all + left_out)) * inv;
    const float r_sum = apart ? warp_sum(f * inv * all) : 0.f, w_sum = warp_sum(f * fmaf(inv * all, dt, q));
    const unsigned int skipped = __reduce_or_sync(~0u, (unsigned int)above) & (unsigned int)kSkipped;
    const int up = __reduce_add_sync(~0u, above & INT_MAX);
    if (lane == 0) {
      if (apart) sh.warp_f[3][warp] = r_sum;
      sh.warp_f[2][warp] = w_sum;
      sh.warp_above[warp] = up | (int)skipped;
    }
    __syncthreads();
    if (k) {
      int n = sh.n;
      if (n > kList)
        n = collect<T>(sh, at.data, at.words, at.index(0), at.x, p.vocab, part ? 0 : head, part ? 0 : tail, k,
                       no_masked());
      rank_keys(sh.list, n, k, sh.sorted);
    }
    Part own{M, 0.f, 0.f, 0};
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      own.r += apart ? sh.warp_f[3][i] : 0.f;
      own.w += sh.warp_f[2][i];
      own.above = ((own.above + sh.warp_above[i]) & INT_MAX) | ((own.above | sh.warp_above[i]) & kSkipped);
    }
    if (!apart) own.r = S - 1.f;  // (NaN: apart is false, and stays NaN)
    if (splits == 1) {
      if (tid == 0) sh.parts[0] = own;
    } else {
      // Into the first CTA's shared memory.
      asm volatile("barrier.cluster.wait;" ::: "memory");  // it has started
      uint32_t to;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(sm100::smem_u32(&sh.parts[part])));
      if (tid == 0)
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(__float_as_uint(own.m)),
                     "r"(__float_as_uint(own.r)), "r"(__float_as_uint(own.w)), "r"(own.above)
                     : "memory");
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(sm100::smem_u32(&sh.gathered[part * k])));
      if (tid < k)
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to + 8 * tid), "l"(sh.sorted[tid]) : "memory");
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      if (part != 0) return;
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      if (k) rank_keys(sh.gathered, splits * k, k, sh.merged);
    }
    __syncthreads();
  }

  // ---- the row
  const int tok = p.token_ids ? p.token_ids[row] : -1;
  const bool has_token = tok >= 0 && tok < p.vocab;
  if (tid == 0 && !has_token && tok != -1 && p.error_bits) atomicOr(p.error_bits, kErrTokenId);
  Part a = splits > 1 ? join(sh.parts, splits) : sh.parts[0];
  if (a.r != a.r || a.w != a.w || a.m > kHighRow || ((a.above & kSkipped) && !(a.m > kLowRow))) {
    general_row<T>(sh, p, at.x, row, head, has_token ? tok : -1);
    return;
  }
  a.above &= INT_MAX;
  u64* top_keys = splits > 1 ? sh.merged : sh.sorted;
  if (k && top_keys[k - 1] == 0) {
    int listed = 0;
    while (top_keys[listed]) ++listed;
    __syncthreads();
    fill_masked<T>(sh, top_keys, at.x, p.vocab, head, listed, k);
  }
  const float nan = __int_as_float(0x7fffffff);
  const float ln_s = a.m == neg_inf() ? nan : log1pf(a.r);
  if (tid == 0) {
    if (p.logprobs) p.logprobs[row] = has_token ? (given - a.m) - ln_s : nan;
    if (p.ranks) p.ranks[row] = has_token ? 1 + a.above : 0;
    if (p.entropy) p.entropy[row] = ln_s - kLn2 * (a.w / (1.f + a.r));
  }
  if (tid < k) {
    const u64 key = top_keys[tid];
    p.top_ids[(long long)row * k + tid] = key_index(key);
    p.top_logprobs[(long long)row * k + tid] = (key_value(key) - a.m) - ln_s;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtas) token_logprobs_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place<T> at(p);
  const uint4* data = at.data + at.first_word();
  const int mine = at.mine(), k = p.num_top;

  auto fill = [&](int from) {  // the warp's tile from word `from` on, by one lane
    const uint32_t bytes = 16u * min(kTileWords, mine - from);
    sm100::mbar_arrive_expect_tx(&sh.full[warp], bytes);
    bulk_load(sh.slot[warp], data + from, bytes, &sh.full[warp]);
  };
  if (lane == 0) {
    sm100::mbar_init(&sh.full[warp], 1);
    sm100::fence_mbar_init();
    if (mine > 0) fill(0);
  }
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const int tok = p.token_ids ? p.token_ids[at.row] : -1;
  float given = __int_as_float(0x7f800000);
  if (k) {
    for (int i = tid; i < kList; i += kThreads) sh.list[i] = 0;
    if (tid < kMaxTop) sh.sorted[tid] = sh.merged[tid] = 0;
    if (tid == 0) {
      sh.n = 0;
      sh.threshold = no_masked();
    }
    if (lane == 0) sh.first_index[warp] = at.index(at.first_word());
  }
  __syncwarp();

  // Per warp: the reference m, rounded to mc in base 2.  Per lane: sums of the tiles since the one that
  // holds m (acc_*), of the tiles before it (s, w) and of that tile itself (p_ref), which is kept
  // apart because it is summed again without m in the end.
  float m = neg_inf(), mc = 0.f, s = 0.f, w = 0.f, p_ref = 0.f;
  u64 acc_s = 0, acc_w = 0;
  int ref_tile = -1;  // its first word (-1: the head and tail logits)
  int above = 0;      // (kSkipped: a bit of it)
  auto flush = [&]() {
    const float2 a = unpack2(acc_s), b = unpack2(acc_w);
    s += a.x + a.y;
    w += b.x + b.y;
    acc_s = acc_w = 0;
  };
  bool lost = false;  // a tile never came: the warp asks for no more, and the row is taken from memory in the end
  for (int from = 0; from == 0 || (from < mine && !lost); from += kTileWords) {
    const int nw = mine - from;  // words from this tile on
    if (nw > 0 && !wait_full(&sh.full[warp], (from / kTileWords) & 1))
      lost = !wait_full(&sh.full[warp], (from / kTileWords) & 1);  // (once more: the copy may be under way)
    // The given logit once a tile has been waited for: it is not waited for alone.
    if (from == 0 && tok >= 0 && tok < p.vocab) given = Elem<T>::load(at.x, tok);
    // A tile lies in registers; of a last one with few words, they are read as they are needed.
    const uint4* slot = sh.slot[warp];
    const bool whole = nw > kTileWords / 2;
    uint4 v[kWords];
    auto word = [&](int u, uint4 (&one)[1]) {
      const int a = lane + u * 32;
      one[0] = a < nw ? slot[a] : make_uint4(Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest, Elem<T>::kLowest);
    };
    float tm = neg_inf();
    if (whole) {
      if (nw >= kTileWords) {
#pragma unroll
        for (int u = 0; u < kWords; ++u) v[u] = slot[lane + u * 32];
      } else {
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
          uint4 one[1];
          word(u, one);
          v[u] = one[0];
        }
      }
      tm = words_max<T>(v);
    } else {
      for (int u = 0; u * 32 < nw; ++u) {
        uint4 one[1];
        word(u, one);
        tm = max_nan(tm, words_max<T>(one));
      }
    }
    const float top = warp_max_nan(tm);

    // ---- candidates
    bool due = false;
    if (k) {
      if (from == 0) {
        // The first threshold: from the top lane maxima of each warp whose lanes all have logits.
        const int full = at.words >= 32 ? min(kWarps, (at.words - 32) / at.share + 1) : 0;
        const int each = full == kWarps ? min(k, 4) : full ? (k + full - 1) / full : 0, all = full * each;
        unsigned int o = tm >= kLow ? order_f32(tm) : 0u;
        if (warp < full) {
          for (int j = 0; j < each; ++j) {
            const unsigned int best = __reduce_max_sync(~0u, o);
            const unsigned int who = __ballot_sync(~0u, o == best);
            if (lane == __ffs(who) - 1) {
              sh.tops[warp * each + j] = best;
              o = 0;
            }
          }
        }
        __syncthreads();
        // The k-th largest of them, in k rounds (all <= 32 then) or by counting.
        unsigned int best = 0;
        if (k <= 8) {
          unsigned int left = lane < all ? sh.tops[lane] : 0u;
          for (int j = 0; j < k && all; ++j) {
            best = __reduce_max_sync(~0u, left);
            const unsigned int who = __ballot_sync(~0u, left == best);
            if (lane == __ffs(who) - 1) left = 0;
          }
        } else {
          for (int j = lane; j < all; j += 32) {
            const unsigned int own = sh.tops[j];
            int larger = 0, least = 0;
#pragma unroll 8
            for (int q = 0; q < all; ++q) {
              larger += sh.tops[q] > own;
              least += sh.tops[q] >= own;
            }
            if (larger < k && k <= least) best = own;
          }
          best = __reduce_max_sync(~0u, best);
        }
        if (best && lane == 0) atomicMax(&sh.threshold, ((u64)best << 32) - 1);
        __syncwarp();
      }
      const float thr_value = value_of_order(reinterpret_cast<volatile unsigned int*>(&sh.threshold)[1]);
      const bool cand = tm >= thr_value;
      if (__any_sync(~0u, cand)) due = list_candidates<T>(sh, from, nw, cand, thr_value, k);
    }
    __syncwarp();  // the slot is read
    if (lane == 0 && from + kTileWords < mine && !lost) fill(from + kTileWords);

    // ---- sums, while the next tiles arrive
    const bool raise = top > m && top >= kLow;
    if (raise) {
      flush();
      move_up(top, m, mc, s, w, p_ref);
      ref_tile = from;
    }
    // A tile far below the reference (banned tokens) adds nothing.
    if (top >= m - 120.f) {
      if (whole) {
        add_words<T>(v, m, mc, acc_s, acc_w);
      } else {
        for (int u = 0; u * 32 < nw; ++u) {
          uint4 one[1];
          word(u, one);
          add_words<T>(one, m, mc, acc_s, acc_w);
        }
      }
    }
    if (top != top) s = top;
    else if (m == neg_inf() && top > neg_inf()) above |= kSkipped;
    if (raise) {
      const float2 a = unpack2(acc_s);
      p_ref = a.x + a.y;
      acc_s = 0;
    }
    if (top > given) {
      if (whole) {
        above += count_above<T>(v, given);
      } else {
        for (int u = 0; u * 32 < nw; ++u) {
          uint4 one[1];
          word(u, one);
          above += count_above<T>(one, given);
        }
      }
    }
    if (due) raise_threshold(sh, k);
  }
  flush();
  if (lost) {
    s = __int_as_float(0x7fffffff);  // as a NaN among the logits does, it sends the row to general_row
    if (lane == 0 && p.error_bits) atomicOr(p.error_bits, kErrTimeout);
  }
  finish<T>(sh, p, m, mc, s, w, p_ref, given, above, ref_tile);
}

// CTAs per row: as many as the GPU's places allow for all rows at once, as long as each has kCtaBytes to read.
// Clusters leave places of a GPC empty that none of them fits into, so that the last few rows before a step run
// after the others (151,936 fp16 logits, no alternatives: 48 rows of 8 CTAs 10.5 us, 53 to 55 of 8 14 us, 56 of 7
// 11.4 us; 80 of 5 12.4 us, 88 of 5 15.2 us, 89 of 4 13.8 us).  From 223 rows on a row is one CTA's: up to 444
// rows, the GPU's places, take about the same time (230 rows 22 us, 444 rows 29 us), and the next row starts a
// second round (445 rows 38 us, 888 rows 52 us).
constexpr int kCtaBytes = 16 * 1024;
static int choose_splits(long long rows, int vocab, int item, int sms) {
  const long long by_size = ((long long)vocab * item + kCtaBytes - 1) / kCtaBytes;
  const long long by_rows = (long long)kCtas * sms / rows;
  const long long s = by_size < by_rows ? by_size : by_rows;
  return s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : (int)s;
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
  NEB_REQUIRE(vocab <= logprobs::kMaxVocab, NEB_ERR_UNSUPPORTED, "rows of more than %d logits are not supported",
              logprobs::kMaxVocab);
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
