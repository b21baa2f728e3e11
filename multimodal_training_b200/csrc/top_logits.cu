// The k largest logits of every row with their ids, in descending order: what a teacher hands to a student.
//
// A logit and its column make one 64-bit key: the logit's bits in an order that integers keep (NaN above everything, as
// torch.topk has it; -0 equal to +0) above the inverted column, so that keys are unique and equal logits go by the lower
// column.  The answer is the k largest keys of the row.
//
// One pass over the row, bound by memory (2048 x 152064 bf16, k = 64: 121 us, 5.1 TB/s).  What is left of the logits is the
// vectors of which an element reaches a lower bound of the k-th largest.  The bound is the k-th largest of what the threads have
// seen as their two sets' largest, which are k different elements; it is raised behind stretches 1, 2, 4, ... of the row, and a
// row in no special order leaves about k (1 + 1 + 1/2 + ...) vectors.  Between those the warps do not wait for one another.  In
// the end the elements of these vectors that reach the last bound, little more than k, are ranked.  (Looking at the elements
// where a vector reaches the bound took as long as the pass itself, 107 -> 226 us for 2048 x 152064 bf16 and k = 64: some lane of
// every third warp's load has one.)  Short rows and large k are bound by the chain of barriers of the bounds and of the ranking.
//
// Where there are too many of them (rising logits, many equal ones) the run is looked at once more, step by step, and the list
// of candidates is cut to its k largest as soon as it fills up; the last of them is the next bound, and columns only grow, so
// equal logits that come later do not reach it.
//
// Few rows are cut into runs of columns, one for each CTA of a cluster; the first CTA ranks the others' lists.
#include "key_range.h"
#include "vocab_rows.cuh"

namespace {

typedef unsigned long long u64;

constexpr int kTopMax = 256;          // largest k
constexpr int kTopSets = 4;           // vectors that a thread loads ahead: one of each set
constexpr int kTopFull = 1024;        // candidates from which on the list is cut
constexpr int kTopCluster = 8;        // most CTAs of a row; their lists fit one list: 8 * 256 = 2048
constexpr int kTopBins = KeyRange::kBins;
constexpr int kTopEdge = 16;          // elements outside whole vectors, at most 7 at each end

template <int kTopThreads>
struct alignas(16) TopShared {
  static constexpr int kVecs = kTopThreads == 128 ? 768 : kTopThreads == 256 ? 1536 : 2048;
  static constexpr int kStep = kTopThreads < 256 ? kTopThreads : 256;      // vectors of a step of the second look
  static constexpr int kList = kTopFull + 8 * kStep;                      // all elements of a step fit behind a list that is not full
  uint4 vec[kVecs];                     // vectors that reach a bound, and which they are
  int vec_at[kVecs];
  alignas(16) u64 list[kList + kTopEdge];
  u64 best[kTopMax];
  int hist[kTopBins], start[kTopBins];
  int digit, need, count;               // of find_digit
  int vecs, taken, kept;
  uint32_t warp_value[2][32];
};

MMT_DEVICE u64 whole_key(uint32_t key, int c) { return (u64)key << 32 | (0xffffffffu - (uint32_t)c); }

// Sum over the lanes up to this one.
MMT_DEVICE int up_to_lane(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}
// Smallest and largest of a block's values, of which each thread has its own smallest and largest.
template <int kTopThreads>
MMT_DEVICE uint2 range_of_block(TopShared<kTopThreads>& s, uint32_t lo, uint32_t hi) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  __syncthreads();
  if (lane == 0) {
    s.warp_value[0][warp] = lo;
    s.warp_value[1][warp] = hi;
  }
  __syncthreads();
  return make_uint2(__reduce_min_sync(0xffffffffu, s.warp_value[0][lane % (kTopThreads / 32)]),
                    __reduce_max_sync(0xffffffffu, s.warp_value[1][lane % (kTopThreads / 32)]));
}
// The bin at which the counts, from the last bin down, reach `need`, how many of it are needed and how many there are, into
// shared memory.  All of the block calls it; the barrier behind it is the caller's.
template <int kTopThreads>
MMT_DEVICE void find_digit(TopShared<kTopThreads>& s, int need) {
  if (threadIdx.x >= 32) return;
  constexpr int kEach = kTopBins / 32;
  // lane l holds the bins from kTopBins - 1 - kEach * l down
  const int from = kTopBins - 1 - kEach * (int)threadIdx.x;
  int mine = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) mine += s.hist[from - j];
  int before = up_to_lane(mine) - mine;          // keys above this lane's bins
  if (before < need && before + mine >= need) {
    int d = from;
    while (before + s.hist[d] < need) before += s.hist[d--];
    s.digit = d;
    s.need = need - before;
    s.count = s.hist[d];
  }
}

// A t that at least k of the block's values, two a thread, reach: near the largest one, the lower end of its bin in a histogram
// of their range above `least` (a t from before) and, 16 bits having 128 values between two powers of two, of eight powers of
// two below the largest value.  `least` if fewer than k values are in that range.
template <int kTopThreads>
MMT_DEVICE uint32_t kth_of_block(TopShared<kTopThreads>& s, const uint32_t (&v)[2], int k, uint32_t least) {
  for (int b = threadIdx.x; b < kTopBins; b += kTopThreads) s.hist[b] = 0;
  if (threadIdx.x == 0) s.digit = -1;
  uint2 r = range_of_block<kTopThreads>(s, min(v[0] - 1u, v[1] - 1u), max(v[0], v[1]));      // 0 is none
  r.x = max(max(r.x + 1u, least), r.y > 1023u ? r.y - 1023u : 1u);
  const int wide = r.y < r.x ? 0 : 32 - __clz((r.y - r.x) / kTopBins);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (v[j] >= r.x) atomicAdd(&s.hist[(v[j] - r.x) >> wide], 1);
  __syncthreads();
  find_digit(s, k);
  __syncthreads();
  return s.digit < 0 ? least : r.x + ((uint32_t)s.digit << wide);
}

// Ranks the n keys of the list and hands out the k largest: out(rank, key).  n >= k, and k of the keys reach `bound` (16 bits
// from `shift` up).  All threads come out of it together.
template <int kTopThreads, typename F>
MMT_DEVICE void rank_list(TopShared<kTopThreads>& s, int n, int k, int shift, uint32_t bound, F out) {
  const int tid = threadIdx.x;
  if (n > k + 64) {                               // what cannot be among the k leaves the list
    uint32_t most = 0;
    for (int i = tid; i < n; i += kTopThreads) most = max(most, (uint32_t)(s.list[i] >> shift) & 0xffffu);
    most = range_of_block<kTopThreads>(s, most, most).y;
    // keys that the range holds compete for `need` places; those above have theirs
    KeyRange range(bound, most, shift);
    int need = k, sure = 0;
    for (;;) {
      for (int b = tid; b < kTopBins; b += kTopThreads) s.hist[b] = 0;
      if (tid == 0) s.kept = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kTopThreads) {
        const u64 key = s.list[i];
        if (range.holds(key)) atomicAdd(&s.hist[range.bin(key)], 1);
      }
      __syncthreads();
      find_digit(s, need);
      __syncthreads();
      range.raise(s.digit);
      sure += need - s.need;
      need = s.need;
      const int left = sure + s.count;
      if (left <= k + 64 || !range.narrow()) break;
      __syncthreads();                            // all have read what find_digit found
    }
    for (int i0 = 0; i0 < n; i0 += kTopThreads) { // in place: what is written has been read
      const u64 key = i0 + tid < n ? s.list[i0 + tid] : 0;
      __syncthreads();
      if (key != 0 && key >= range.low) s.list[atomicAdd(&s.kept, 1)] = key;
      __syncthreads();
    }
    n = s.kept;
  }
  // At most k + 64 keys are left.  They go into 256 bins of their values, and a key's rank is what lies in the bins above plus
  // the larger ones of its own bin.  (4096 x 2000 fp32 and k = 256: 61 us; 103 when the larger ones of all were counted.)
  constexpr int kEach = (kTopMax + 64 + kTopThreads - 1) / kTopThreads;
  u64 key[kEach];
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    key[e] = tid + e * kTopThreads < n ? s.list[tid + e * kTopThreads] : 0;
    if (key[e] != 0) {
      lo = min(lo, (uint32_t)(key[e] >> 32));
      hi = max(hi, (uint32_t)(key[e] >> 32));
    }
  }
  for (int b = tid; b < kTopBins; b += kTopThreads) s.hist[b] = 0;
  const uint2 range = range_of_block<kTopThreads>(s, lo, hi);
  const int wide = range.y < range.x ? 0 : 32 - __clz((range.y - range.x) / kTopBins);
  int bin[kEach], at[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    bin[e] = key[e] != 0 ? (int)(((uint32_t)(key[e] >> 32) - range.x) >> wide) : -1;
    if (bin[e] >= 0) at[e] = atomicAdd(&s.hist[bin[e]], 1);
  }
  __syncthreads();
  if (tid < 32) {                                 // where the bins' keys start, from the last bin down
    constexpr int kLane = kTopBins / 32;
    const int from = kTopBins - 1 - kLane * tid;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kLane; ++j) mine += s.hist[from - j];
    int before = up_to_lane(mine) - mine;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      s.start[from - j] = before;
      before += s.hist[from - j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (bin[e] >= 0) s.list[s.start[bin[e]] + at[e]] = key[e];
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (bin[e] < 0) continue;
    int rank = s.start[bin[e]];
    const int end = rank + s.hist[bin[e]];
    for (int j = rank; j < end; ++j) rank += s.list[j] > key[e];
    if (rank < k) out(rank, key[e]);
  }
  __syncthreads();
}

template <typename T, int kTopThreads>
__global__ void __launch_bounds__(kTopThreads, 1024 / kTopThreads) top_logits_kernel(const T* logits, T* __restrict__ values,
                                                                                    long* __restrict__ ids, int V, long ld,
                                                                                    int k, long vocab_lo, int per) {
  grid_dependency_sync();
  constexpr int kStretch = kTopSets * kTopThreads, kVec = Row<T>::kVec;
  constexpr int kVecs = TopShared<kTopThreads>::kVecs, kStep = TopShared<kTopThreads>::kStep;
  constexpr int kList = TopShared<kTopThreads>::kList;
  extern __shared__ __align__(128) uint4 shared[];
  TopShared<kTopThreads>& s = *reinterpret_cast<TopShared<kTopThreads>*>(shared);
  const int tid = threadIdx.x;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const long r = blockIdx.x / C;
  // vectors [first, stop) of the row, whole ones [lo, hi)
  const Row<T> row(logits + r * ld, V);
  const int first = rank * per, stop = min(first + per, row.vectors());
  const int lo = first + (first == 0 && row.lead != 0), hi = min(stop, (row.lead + V) / Row<T>::kVec);
  // how many of the k this run may hold
  auto most_of = [&](int q) {
    const int from = max(row.column(q * per), 0), to = min(row.column(min((q + 1) * per, row.vectors())), V);
    return min(k, max(to - from, 0));
  };
  const int mine_k = most_of(rank);
  uint4 next[kTopSets];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kTopSets; ++j) {
      const int i = i0 + j * kTopThreads + tid;
      if (i < hi) next[j] = *reinterpret_cast<const uint4*>(row.p + row.column(i));
    }
  };
  load(lo);
  if (tid == 0) s.taken = s.vecs = 0;
  __syncthreads();
  constexpr int kDrop = Key<T>::kBits - 16, kShift = 32 + kDrop;
  // a key below `least` is not among the k; k of the logits looked at so far reach the 16 bits of `bound`; `top` are 16 bits of
  // this thread's largest of the even and the odd sets
  uint32_t least = 0, bound = 0, top[2] = {0, 0};
  auto push = [&](uint32_t key, int c) {            // whether the list is full
    if (key < least) return false;
    const int at = atomicAdd(&s.taken, 1);
    if (at < kList + kTopEdge) s.list[at] = whole_key(key, c);
    return at + 1 >= kTopFull;
  };
  // elements in front of the first whole vector, and behind the last one
  auto push_edge = [&](int from, int to) {
    if (from + tid < to) push(Key<T>::of(row.p[from + tid]), from + tid);
  };
  const int head = max(row.column(first), 0), head_end = min(row.column(min(lo, stop)), V);
  int look = 1;
  bool over = false;
  for (int i0 = lo, n = 1; i0 < hi && !over; i0 += kStretch, ++n) {
    uint4 u[kTopSets];
    uint32_t t[kTopSets];
#pragma unroll
    for (int j = 0; j < kTopSets; ++j) u[j] = next[j];
    load(i0 + kStretch);
#pragma unroll
    for (int j = 0; j < kTopSets; ++j) {
      t[j] = i0 + j * kTopThreads + tid < hi ? Key<T>::top16(u[j]) : 0;
      top[j % 2] = max(top[j % 2], t[j]);
    }
    if (n == look) {
      bound = kth_of_block<kTopThreads>(s, top, k, bound);
      over = __syncthreads_or(s.vecs > kVecs);
      look *= 2;
    }
#pragma unroll
    for (int j = 0; j < kTopSets; ++j)
      if (t[j] >= max(bound, 1u)) {
        const int at = atomicAdd(&s.vecs, 1);
        if (at < kVecs) {
          s.vec[at] = u[j];
          s.vec_at[at] = i0 + j * kTopThreads + tid;
        }
      }
  }
  __syncthreads();
  uint32_t listed = bound;                          // k of the keys in the list reach it (all, as long as there are fewer)
  least = bound << kDrop;
  const int vecs = s.vecs;
  if (vecs <= kVecs) {
    push_edge(head, head_end);
    for (int q = tid; q < vecs * kVec; q += kTopThreads) {
      const T x = reinterpret_cast<const T*>(s.vec)[q];
      push(Key<T>::of(x), row.column(s.vec_at[q / kVec]) + q % kVec);
    }
  }
  __syncthreads();
  if (vecs > kVecs || s.taken > kList) {
    __syncthreads();
    if (tid == 0) s.taken = 0;
    least = listed = 0;
    __syncthreads();
    push_edge(head, head_end);
    for (int i0 = lo; i0 < hi; i0 += kStep) {
      const int i = i0 + tid;
      bool full = false;
      if (tid < kStep && i < hi) {
        const uint4 u = *reinterpret_cast<const uint4*>(row.p + row.column(i));
        if (Key<T>::top16(u) >= least >> kDrop) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) full |= push(Key<T>::of(element<T>(u, e)), row.column(i) + e);
        }
      }
      if (!__syncthreads_or(full)) continue;        // seen by the threads that took those places: the same for all
      rank_list<kTopThreads>(s, s.taken, k, kShift, listed, [&](int at, u64 key) { s.best[at] = key; });
      for (int q = tid; q < k; q += kTopThreads) s.list[q] = s.best[q];
      listed = (uint32_t)(s.best[k - 1] >> kShift);
      least = (uint32_t)(s.best[k - 1] >> 32) + 1;
      if (tid == 0) s.taken = k;
      __syncthreads();
    }
  }
  __syncthreads();
  push_edge(max(row.column(max(hi, lo)), 0), min(row.column(stop), V));
  __syncthreads();
  const int n = s.taken;
  auto answer = [&](int at, u64 key) {
    const uint32_t c = 0xffffffffu - (uint32_t)key;
    T x;
    // zeros and NaN have lost bits in their keys
    if (!Key<T>::back((uint32_t)(key >> 32), x)) x = row.p[c];
    values[r * k + at] = x;
    ids[r * k + at] = vocab_lo + c;
  };
  if (C == 1) {
    rank_list<kTopThreads>(s, n, k, kShift, listed, answer);
    return;
  }
  rank_list<kTopThreads>(s, n, mine_k, kShift, listed, [&](int at, u64 key) { s.best[at] = key; });
  cluster_barrier();                                // every CTA has its list
  if (rank == 0) {
    // behind one another, in the order of the CTAs; a list of k ends at a bound of the whole row's k-th largest
    int at = 0;
    listed = 0;
    for (int q = 0; q < C; ++q) {
      const int q_k = most_of(q);
      for (int i = tid; i < q_k; i += kTopThreads) s.list[at + i] = cluster_load(&s.best[i], q);
      if (q_k == k) listed = max(listed, (uint32_t)(cluster_load(&s.best[k - 1], q) >> kShift));
      at += q_k;
    }
    __syncthreads();
    rank_list<kTopThreads>(s, at, k, kShift, listed, answer);
  }
  cluster_barrier();                                // the first CTA has read the lists
}

template <typename T, int kTopThreads>
int launch_threads(const void* logits, void* values, long* ids, long rows, int V, long ld, int k, long vocab_lo, int C, int per,
                   void* stream) {
  auto kernel = top_logits_kernel<T, kTopThreads>;
  constexpr size_t kBytes = sizeof(TopShared<kTopThreads>);
  static bool allowed = false;
  if (!allowed) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBytes);
    if (e != cudaSuccess) return (int)e;
    allowed = true;
  }
  return (int)launch_cluster(kernel, (unsigned)(rows * C), kTopThreads, C, kBytes, VR_STREAM(stream),
                             reinterpret_cast<const T*>(logits), reinterpret_cast<T*>(values), ids, V, ld, k, vocab_lo, per);
}
template <typename T>
int launch_top(const void* logits, void* values, long* ids, long rows, int V, long ld, int k, long vocab_lo,
               void* stream) {
  const long nv = ((long)V + Row<T>::kVec - 2) / Row<T>::kVec + 1;
  // few rows: up to two CTAs an SM, as long as a CTA has a vector for each thread
  int C = 1;
  while (C < kTopCluster && rows * C * 2 <= 2L * mmt_sm_count() && nv > 512L * C) C *= 2;
  const int per = (int)((nv + C - 1) / C);
  // Short rows have few stretches, and more of them fit an SM in smaller CTAs; a large k needs many values for its bound.
  // us with 128, 256 and 512 threads, 4096 rows in bf16: 5000 columns 33, 42, 60 (k = 64) and 97, 72, 88 (k = 256); 16000 columns
  // 48, 57, 64 (k = 32) and 248, 101, 87 (k = 256); 2048 x 50000 and k = 32: 56, 54, 63; 1024 x 152064 and k = 256: 424, 172, 83.
  if (C == 1 && k <= 64 && per <= 2048)
    return launch_threads<T, 128>(logits, values, ids, rows, V, ld, k, vocab_lo, C, per, stream);
  return C == 1 && per <= (k <= 64 ? 8192 : 1024)
             ? launch_threads<T, 256>(logits, values, ids, rows, V, ld, k, vocab_lo, C, per, stream)
             : launch_threads<T, 512>(logits, values, ids, rows, V, ld, k, vocab_lo, C, per, stream);
}

}  // namespace

extern "C" {

// values [rows, k] in the logits' type and ids [rows, k]; 1 <= k <= min(V, 256), one stride of `ld` elements between rows.
int mmt_top_logits(const void* logits, int is_f32, void* values, long* ids, long rows, int V, long ld, int k, long vocab_lo,
                   void* stream) {
  if (k < 1 || k > kTopMax || k > V || rows > 0x7fffffffL / kTopCluster) return -2;
  if (rows == 0) return 0;
  return is_f32 ? launch_top<float>(logits, values, ids, rows, V, ld, k, vocab_lo, stream)
                : launch_top<bf16>(logits, values, ids, rows, V, ld, k, vocab_lo, stream);
}

}  // extern "C"
