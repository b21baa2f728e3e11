// The k largest logits of every row with their ids, in descending order: what a teacher hands to a student.
//
// A logit and its column make one 64-bit key: the logit's bits in an order that integers keep (NaN above everything, as
// torch.topk has it; -0 equal to +0) above the inverted column, so that keys are unique and equal logits go by the lower
// column.  The answer is the k largest keys of the row.
//
// One CTA per row.  The k-th largest logit is found digit by digit (8 bits, most significant first) from histograms of
// the row; a last pass collects what lies above it and, in the order of the columns, as many of its equals as are needed.
#include "vocab_rows.cuh"

namespace {

typedef unsigned long long u64;

constexpr int kTopThreads = 512;
constexpr int kTopMax = 256;          // largest k

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
};

// Calls f(key, column) for every element of vector i that the row has.
template <typename T, typename F>
MMT_DEVICE void each_key(const Row<T>& row, int i, F f) {
  const uint4 u = row.load(i);
  const T* e = reinterpret_cast<const T*>(&u);
  const int c = row.column(i);
#pragma unroll
  for (int j = 0; j < Row<T>::kVec; ++j)
    if (c + j >= 0 && c + j < row.V) f(Key<T>::of(e[j]), c + j);
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads) top_logits_kernel(const T* logits, T* __restrict__ values,
                                                                 long* __restrict__ ids, int V, long ld, int k,
                                                                 long vocab_lo) {
  grid_dependency_sync();
  __shared__ int hist[256];
  __shared__ int found[3];                       // digit, how many of it are needed, how many there are
  __shared__ int taken;
  __shared__ int warp_count[kTopThreads / 32];
  __shared__ u64 best[kTopMax];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Row<T> row(logits + blockIdx.x * ld, V);
  const int nv = row.vectors();

  uint32_t prefix = 0, mask = 0;
  int need = k;
  for (int shift = Key<T>::kBits - 8; shift >= 0; shift -= 8) {
    for (int b = tid; b < 256; b += kTopThreads) hist[b] = 0;
    __syncthreads();
    for (int i = tid; i < nv; i += kTopThreads)
      each_key<T>(row, i, [&](uint32_t key, int) {
        if ((key & mask) == prefix) atomicAdd(&hist[key >> shift & 255u], 1);
      });
    __syncthreads();
    if (warp == 0) {
      // lane l holds the eight digits from 255 - 8 l down
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) mine += hist[255 - 8 * lane - j];
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= mine;                            // keys above this lane's digits
      if (before < need && before + mine >= need) {
        int d = 255 - 8 * lane;
        while (before + hist[d] < need) before += hist[d--];
        found[0] = d;
        found[1] = need - before;
        found[2] = hist[d];
      }
    }
    if (tid == 0) taken = 0;
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    mask |= 255u << shift;
    need = found[1];
  }
  const bool all_ties = found[2] == need;
  for (int i = tid; i < nv; i += kTopThreads)
    each_key<T>(row, i, [&](uint32_t key, int c) {
      if (key > prefix || (all_ties && key == prefix))
        best[atomicAdd(&taken, 1)] = (u64)key << 32 | (0xffffffffu - (uint32_t)c);
    });
  __syncthreads();
  if (!all_ties) {
    // the lowest columns among equals: whole blocks of vectors in the order of the columns
    int place = taken;
    for (int i0 = 0; i0 < nv && place < k; i0 += kTopThreads) {
      int mine = 0;
      if (i0 + tid < nv) each_key<T>(row, i0 + tid, [&](uint32_t key, int) { mine += key == prefix; });
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      if (lane == 31) warp_count[warp] = before;
      before -= mine;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < kTopThreads / 32; ++w) {
        before += w < warp ? warp_count[w] : 0;
        total += warp_count[w];
      }
      int at = place + before;
      if (mine && at < k)
        each_key<T>(row, i0 + tid, [&](uint32_t key, int c) {
          if (key == prefix && at < k) best[at++] = (u64)key << 32 | (0xffffffffu - (uint32_t)c);
        });
      place += total;
      __syncthreads();
    }
  }
  if (tid < k) {
    const u64 mine = best[tid];
    int rank = 0;
    for (int j = 0; j < k; ++j) rank += best[j] > mine;
    const uint32_t c = 0xffffffffu - (uint32_t)mine;
    values[blockIdx.x * (long)k + rank] = row.p[c];
    ids[blockIdx.x * (long)k + rank] = vocab_lo + c;
  }
}

template <typename T>
int launch_top(const void* logits, void* values, long* ids, long rows, int V, long ld, int k, long vocab_lo,
               void* stream) {
  return (int)launch_dependent(top_logits_kernel<T>, (unsigned)rows, kTopThreads, 0, VR_STREAM(stream),
                               reinterpret_cast<const T*>(logits), reinterpret_cast<T*>(values), ids, V, ld, k, vocab_lo);
}

}  // namespace

extern "C" {

// values [rows, k] in the logits' type and ids [rows, k]; 1 <= k <= min(V, 256), one stride of `ld` elements between rows.
int mmt_top_logits(const void* logits, int is_f32, void* values, long* ids, long rows, int V, long ld, int k, long vocab_lo,
                   void* stream) {
  if (k < 1 || k > kTopMax || k > V || rows > 0x7fffffffL) return -2;
  if (rows == 0) return 0;
  return is_f32 ? launch_top<float>(logits, values, ids, rows, V, ld, k, vocab_lo, stream)
                : launch_top<bf16>(logits, values, ids, rows, V, ld, k, vocab_lo, stream);
}

}  // extern "C"
