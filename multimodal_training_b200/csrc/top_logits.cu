// The k largest logits of every row with their ids, in descending order: what a teacher hands to a student.
//
// A logit and its column make one 64-bit key: the logit's bits in an order that integers keep (NaN above everything, as
// torch.topk has it; -0 equal to +0) above the inverted column, so that keys are unique and equal logits go by the lower
// column.  The answer is the k largest keys of the row.
//
// One pass over the row, bound by memory: what is left of each stretch of logits is what reaches a lower bound of the k-th
// largest logit.  The bound is the k-th largest of the threads' own largest logits, which are k different elements; a row in
// no special order leaves about k (1 + 1 + 1/2 + ...) candidates.  They are ranked by counting.  Rows in rising order, or
// with many equal logits, overflow the list of candidates; such a row is selected digit by digit from histograms instead,
// with further passes over it.
//
// Few rows are cut into runs of columns, one for each CTA of a cluster; the first CTA ranks the others' lists.
#include "vocab_rows.cuh"

namespace {

typedef unsigned long long u64;

constexpr int kTopThreads = 512;
constexpr int kTopWarps = kTopThreads / 32;
constexpr int kTopMax = 256;          // largest k
constexpr int kTopList = 2048;        // candidates that are kept
constexpr int kTopAhead = 4;          // vectors that a thread loads before it looks at them
constexpr int kTopCluster = 8;        // most CTAs of a row; their lists fit one list: 8 * 256 = 2048

// Order-preserving bits of a logit; kBits of them.
template <typename T>
struct Key;
template <>
struct Key<bf16> {
  static constexpr int kBits = 16;
  static MMT_DEVICE uint32_t of(bf16 x) {
    uint32_t b = __bfloat16_as_ushort(x);
    if ((b & 0x7fffu) > 0x7f80u) return 0xffffu;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
  }
  // Bits of the largest element of a vector that bound a thread's largest from below, as of() orders them; 16 of them.
  static MMT_DEVICE uint32_t top16(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) t = __hmax2_nan(t, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    return of(__hmax_nan(__low2bfloat16(t), __high2bfloat16(t)));
  }
};
template <>
struct Key<float> {
  static constexpr int kBits = 32;
  static MMT_DEVICE uint32_t of(float x) {
    uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if (b == 0x80000000u) b = 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static MMT_DEVICE uint32_t top16(const uint4& u) {
    const float v[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w)};
    uint32_t t = of(v[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) t = max(t, of(v[j]));
    return t >> 16;
  }
};

// A CTA's run of a row: vectors [first, stop).
template <typename T>
struct Run {
  Row<T> row;
  int first, stop;
};

struct TopShared {
  u64 list[kTopList];
  u64 best[kTopMax];
  int hist[256];
  int found[3];
  int taken, kept;
  int warp_count[kTopWarps];
};

// Calls f(key, column) for every element of vector i that the row has.
template <typename T, typename F>
MMT_DEVICE void each_key(const Row<T>& row, int i, const uint4& u, F f) {
  const T* e = reinterpret_cast<const T*>(&u);
  const int c = row.column(i);
#pragma unroll
  for (int j = 0; j < Row<T>::kVec; ++j)
    if (c + j >= 0 && c + j < row.V) f(Key<T>::of(e[j]), c + j);
}
template <typename T, typename F>
MMT_DEVICE void each_key(const Row<T>& row, int i, F f) {
  each_key<T>(row, i, row.load(i), f);
}
MMT_DEVICE u64 whole_key(uint32_t key, int c) { return (u64)key << 32 | (0xffffffffu - (uint32_t)c); }

// The largest t of 16 bits that at least k of the block's values reach (0 if there are fewer than k).  A thread has N
// values, of which the first `n` (the same for all threads) count.
template <int N>
MMT_DEVICE uint32_t kth_of_block(const uint32_t (&v)[N], int n, int k) {
  uint32_t t = 0;
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t at = t | 1u << bit;
    int count = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) count += __syncthreads_count(v[j] >= at);
    if (count >= k) t = at;
  }
  return t;
}

// best[0, k) := the k largest keys of a run that has at least k elements, in no order.  Digits of 8 bits from histograms.
template <typename T>
MMT_DEVICE void select_by_digits(const Run<T>& run, int k, TopShared& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Row<T>& row = run.row;
  uint32_t prefix = 0, mask = 0;
  int need = k;
  for (int shift = Key<T>::kBits - 8; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int b = tid; b < 256; b += kTopThreads) s.hist[b] = 0;
    __syncthreads();
    for (int i = run.first + tid; i < run.stop; i += kTopThreads)
      each_key<T>(row, i, [&](uint32_t key, int) {
        if ((key & mask) == prefix) atomicAdd(&s.hist[key >> shift & 255u], 1);
      });
    __syncthreads();
    if (warp == 0) {
      // lane l holds the eight digits from 255 - 8 l down
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) mine += s.hist[255 - 8 * lane - j];
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= mine;                            // keys above this lane's digits
      if (before < need && before + mine >= need) {
        int d = 255 - 8 * lane;
        while (before + s.hist[d] < need) before += s.hist[d--];
        s.found[0] = d;
        s.found[1] = need - before;
        s.found[2] = s.hist[d];
      }
    }
    if (tid == 0) s.taken = 0;
    __syncthreads();
    prefix |= (uint32_t)s.found[0] << shift;
    mask |= 255u << shift;
    need = s.found[1];
  }
  const bool all_ties = s.found[2] == need;
  for (int i = run.first + tid; i < run.stop; i += kTopThreads)
    each_key<T>(row, i, [&](uint32_t key, int c) {
      if (key > prefix || (all_ties && key == prefix)) s.best[atomicAdd(&s.taken, 1)] = whole_key(key, c);
    });
  __syncthreads();
  if (all_ties) return;
  // the lowest columns among equals: whole blocks of vectors in the order of the columns
  int place = s.taken;
  for (int i0 = run.first; i0 < run.stop && place < k; i0 += kTopThreads) {
    int mine = 0;
    if (i0 + tid < run.stop) each_key<T>(row, i0 + tid, [&](uint32_t key, int) { mine += key == prefix; });
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    if (lane == 31) s.warp_count[warp] = before;
    before -= mine;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kTopWarps; ++w) {
      before += w < warp ? s.warp_count[w] : 0;
      total += s.warp_count[w];
    }
    int at = place + before;
    if (mine && at < k)
      each_key<T>(row, i0 + tid, [&](uint32_t key, int c) {
        if (key == prefix && at < k) s.best[at++] = whole_key(key, c);
      });
    place += total;
    __syncthreads();
  }
}

// Ranks the n keys of the list that reach `bound` (16 bits of a logit's order) and hands out the k largest: out(rank, key).
// At least k do.  `shift`: of the 16 bits in a key.
template <typename F>
MMT_DEVICE void rank_list(TopShared& s, int n, int k, int shift, F out) {
  const int tid = threadIdx.x;
  constexpr int kEach = kTopList / kTopThreads;
  u64 mine[kEach];
  uint32_t v[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = tid + j * kTopThreads;
    mine[j] = i < n ? s.list[i] : 0;
    v[j] = (uint32_t)(mine[j] >> shift) & 0xffffu;
  }
  if (n > 64) {                                     // what cannot be among the k leaves the list
    const uint32_t t = kth_of_block(v, (n + kTopThreads - 1) / kTopThreads, k);
    if (tid == 0) s.kept = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (mine[j] != 0 && v[j] >= t) s.list[atomicAdd(&s.kept, 1)] = mine[j];
    __syncthreads();
    n = s.kept;
  }
  for (int i = tid; i < n; i += kTopThreads) {
    const u64 key = s.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.list[j] > key;
    if (rank < k) out(rank, key);
  }
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 3) top_logits_kernel(const T* logits, T* __restrict__ values,
                                                                    long* __restrict__ ids, int V, long ld, int k,
                                                                    long vocab_lo, int per) {
  grid_dependency_sync();
  __shared__ TopShared s;
  const int tid = threadIdx.x;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const long r = blockIdx.x / C;
  Run<T> run = {Row<T>(logits + r * ld, V), rank * per, 0};
  run.stop = min(run.first + per, run.row.vectors());
  // elements of this run, and how many of them may be among the k
  const int lo = max(run.row.column(run.first), 0), hi = min(run.row.column(run.stop), V);
  const int mine_k = min(k, max(hi - lo, 0));
  if (tid == 0) s.taken = 0;
  __syncthreads();
  uint32_t bound = 0, top[1] = {0};                 // 16 bits of the k-th largest's lower bound, of this thread's largest
  bool over = false;
  int look = 1;                                     // stretches behind which the bound is raised: 1, 2, 4, ...
  for (int i0 = run.first, n = 0; i0 < run.stop && !over; i0 += kTopAhead * kTopThreads, ++n) {
    uint4 u[kTopAhead];
    uint32_t t[kTopAhead];
#pragma unroll
    for (int j = 0; j < kTopAhead; ++j) {
      const int i = i0 + j * kTopThreads + tid;
      t[j] = 0;
      if (i < run.stop) u[j] = run.row.load(i);
    }
#pragma unroll
    for (int j = 0; j < kTopAhead; ++j) {
      if (i0 + j * kTopThreads + tid < run.stop) t[j] = Key<T>::top16(u[j]);
      top[0] = max(top[0], t[j]);
    }
    if (n + 1 == look) {
      bound = kth_of_block(top, 1, k);
      look *= 2;
    }
#pragma unroll
    for (int j = 0; j < kTopAhead; ++j) {
      const int i = i0 + j * kTopThreads + tid;
      if (i < run.stop && t[j] >= bound)
        each_key<T>(run.row, i, u[j], [&](uint32_t key, int c) {
          if (key >> (Key<T>::kBits - 16) >= bound) {
            const int at = atomicAdd(&s.taken, 1);
            if (at < kTopList) s.list[at] = whole_key(key, c);
          }
        });
    }
    // every stretch ends together only where the bound is raised; an overflow shows at the latest behind the last
    if (n + 1 == look - 1 || n % 4 == 3) over = __syncthreads_or(s.taken > kTopList);
  }
  __syncthreads();
  if (s.taken > kTopList) {
    select_by_digits<T>(run, mine_k, s);
    __syncthreads();
    if (tid < mine_k) s.list[tid] = s.best[tid];
    if (tid == 0) s.taken = mine_k;
    __syncthreads();
  }
  const int n = s.taken;
  constexpr int kShift = 32 + Key<T>::kBits - 16;
  auto answer = [&](int at, u64 key) {
    const uint32_t c = 0xffffffffu - (uint32_t)key;
    values[r * k + at] = run.row.p[c];
    ids[r * k + at] = vocab_lo + c;
  };
  if (C == 1) {
    rank_list(s, n, k, kShift, answer);
    return;
  }
  rank_list(s, n, mine_k, kShift, [&](int at, u64 key) { s.best[at] = key; });
  __syncthreads();
  cluster_barrier();                                // every CTA has its list
  if (rank == 0) {
    // behind one another, in the order of the CTAs
    int at = 0;
    for (int q = 0; q < C; ++q) {
      const int q_lo = max(run.row.column(q * per), 0), q_hi = min(run.row.column(min((q + 1) * per, run.row.vectors())), V);
      const int q_k = min(k, max(q_hi - q_lo, 0));
      if (tid < q_k) s.list[at + tid] = cluster_load(&s.best[tid], q);
      at += q_k;
    }
    __syncthreads();
    rank_list(s, at, k, kShift, answer);
  }
  cluster_barrier();                                // the first CTA has read the lists
}

template <typename T>
int launch_top(const void* logits, void* values, long* ids, long rows, int V, long ld, int k, long vocab_lo,
               void* stream) {
  // two thirds of a wave or more: a CTA for each row; below that as many as keep a stretch of vectors each
  const long nv = ((long)V + Row<T>::kVec - 2) / Row<T>::kVec + 1;
  int C = 1;
  while (C < kTopCluster && rows * C * 2 <= 3L * mmt_sm_count() && nv > (long)kTopThreads * C) C *= 2;
  const int per = (int)((nv + C - 1) / C);
  return (int)launch_cluster(top_logits_kernel<T>, (unsigned)(rows * C), kTopThreads, C, 0, VR_STREAM(stream),
                             reinterpret_cast<const T*>(logits), reinterpret_cast<T*>(values), ids, V, ld, k, vocab_lo, per);
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
