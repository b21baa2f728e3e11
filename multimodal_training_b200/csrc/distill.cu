// Distillation from a teacher's top logits: loss and gradient of a student's logits.
//
//   p = softmax over the kept ids of teacher / tau         q  = softmax over the vocabulary of logits / tau
//   row loss = (1 - a) tau^2 sum_j p_j (log p_j - log q_{id_j}) / N_t  +  a (-log q1_label) / N_l,   q1 = softmax(logits)
//   row gradient = (1 - a) tau / N_t (q_v - sum_{j: id_j = v} p_j)  +  a / N_l (q1_v - [v = label])
//
// N_t counts the rows with a teacher, N_l those with a label; a row without either has no loss and a gradient of zero, and
// its logits are not read.  The vocabulary may be one shard of several: the statistics of a row are then reduced over the
// ranks between the kernels.
//
// Powers of two: with c = log2(e) / tau rounded to fp32 and m the row's largest logit, q_v = 2^((x_v - m) c) / S,
// S = sum 2^((x - m) c).  Statistics and gradient use the same rounded c, which changes the temperature by 2^-24 and nothing
// else; the difference is taken first, so any finite logits do, the lowest of their type among them.  S is summed in fp32: a
// power is off by 2^-22, and a thread adds its terms one by one, up to 200 of them where a cluster holds the row and V / 512
// in the other kernels, each time 2^-24 at most (gradients of 777 x 50001 fp32 logits are off by less than 2^-22 of their
// norm).  The teacher's probabilities are rounded to fp32; sums over the K of them are fp64.
#include <numeric>

#include "vocab_rows.cuh"

namespace {

constexpr int kMaxTop = 256;              // most teacher logits of a row
constexpr int kDistillThreads = 512;
constexpr double kLn2 = 0.69314718055994530942;

// What a row has (DistillRows::mark): kTaught, kLabelled, and the label's slot above them.
constexpr int kTaught = 1, kLabelled = 2, kSlotShift = 2;

// The teacher's side of a batch, K + 1 slots a row: ids without repeats (the first K in the teacher's order, an unused
// slot has id -1; the last one holds the label if the teacher has not), their probabilities, and per row
// info = (sum p log p, sum of the probabilities as rounded).  counts: rows with a teacher / with a label, per block.
struct DistillRows {
  int* slot_id;
  float* slot_p;
  double2* info;
  int* mark;
  int2* counts;
  int K, n_counts;
};

// Scalars of a call.
struct DistillCall {
  float c, c1;                            // log2(e) / tau and log2(e)
  float temperature, share;
};

// Per row, in statistics of [kStats][rows], of this shard: m c and m c1, S and S1, (x - m) c1 of the label if it is here and
// 1 then, sum of p (x - m) c and of p over the slots that are here; and the row's loss, for which further backward passes
// leave the others as they are.  Or parts of the row's loss, one from each CTA that has worked on it, which start as zeros.
constexpr int kMaxCluster = 8;
enum { kTop, kTop1, kSum, kSum1, kLabel, kDot, kMass, kMine, kLoss, kStats };
static_assert(kStats >= kMaxCluster, "the parts of a row's loss lie where its statistics do");

// ----------------------------------------------------------------------------
// Teacher's side: one warp per row.  An entry is absent if its id is negative or its logit -inf.  2048 rows of 64: 9 us, a
// chain of fp64 exponentials and of 16 comparisons a lane for repeated ids.
// ----------------------------------------------------------------------------
constexpr int kPrepareRows = 8;                    // warps of a block
template <typename T>
__global__ void __launch_bounds__(32 * kPrepareRows) distill_prepare_kernel(const long* ids, long ids_ld, const T* teacher,
                                                                            long teacher_ld, const long* labels, long rows,
                                                                            long vocab, double inv_temperature, int taught,
                                                                            DistillRows out, long* need,
                                                                            double* stats, int* ticket,
                                                                            MmtErrorWord* ew) {
  grid_dependency_sync();
  __shared__ __align__(16) int s_id[kPrepareRows][kMaxTop];
  __shared__ double s_p[kPrepareRows][kMaxTop];
  __shared__ int marks[kPrepareRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = out.K;
  const long row = (long)blockIdx.x * kPrepareRows + warp;
  if (blockIdx.x == 0 && threadIdx.x == 0) ticket[0] = ticket[1] = 0;
  int mark = 0;
  if (row < rows) {
    double top = -INFINITY;
    bool any = false, odd = false;                  // odd: a logit that is not a number
    for (int j = lane; j < (K + 3) / 4 * 4; j += 32) {
      long id = -1;
      float t = -INFINITY;
      if (j < K) {
        id = ids[row * ids_ld + j];
        t = to_float(teacher[row * teacher_ld + j]);
      }
      if (id >= vocab) {
        mmt_report(ew, MMT_ERR_BOUNDS, 700, (int)row);
        id = -1;
      }
      const bool here = taught && id >= 0 && !(t == -INFINITY);
      s_id[warp][j] = here ? (int)id : -1;
      s_p[warp][j] = here ? (double)t * inv_temperature : -INFINITY;
      any |= here;
      odd |= here && !(t == t);
      if (here) top = fmax(top, (double)t * inv_temperature);
    }
    any = __any_sync(0xffffffffu, any);
    odd = __any_sync(0xffffffffu, odd);
    double total = 0.0, dot = 0.0;
    if (any) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (odd) top = NAN;
      for (int j = lane; j < K; j += 32)
        if (s_id[warp][j] >= 0) {
          const double z = s_p[warp][j] - top, e = exp(z);
          s_p[warp][j] = e;
          total += e;
          if (!(e == 0.0)) dot += e * z;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
    }
    __syncwarp();
    long label = labels ? labels[row] : -1;
    if (label >= vocab) {
      if (lane == 0) mmt_report(ew, MMT_ERR_BOUNDS, 701, (int)row);
      label = -1;
    }
    // an id that the teacher gives more than once has the sum of its probabilities, in the first of its slots
    double sum_p = 0.0;
    int at_label = K;
    const double inv_total = any ? 1.0 / total : 0.0;
    for (int j = lane; j < K; j += 32) {
      const int id = any ? s_id[warp][j] : -1;
      float rounded = 0.f;
      bool first = id >= 0;
      if (first) {
        int same = 0, before = 0;
        for (int i = 0; i < K; i += 4) {
          const int4 q = *reinterpret_cast<const int4*>(&s_id[warp][i]);
          const int hits = (q.x == id) | (q.y == id) << 1 | (q.z == id) << 2 | (q.w == id) << 3;
          same += __popc(hits);
          if (i < j) before |= j - i >= 4 ? hits : hits & ((1 << (j - i)) - 1);
        }
        first = before == 0;
        if (first) {
          double p = s_p[warp][j];
          if (same > 1)
            for (int i = j + 1; i < K; ++i) p += s_id[warp][i] == id ? s_p[warp][i] : 0.0;
          rounded = (float)(p * inv_total);
        }
      }
      out.slot_id[row * (K + 1) + j] = first ? id : -1;
      out.slot_p[row * (K + 1) + j] = rounded;
      sum_p += (double)rounded;
      if (first && id == label) at_label = j;
    }
    if (any) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum_p += __shfl_xor_sync(0xffffffffu, sum_p, o);
    }
    at_label = __reduce_min_sync(0xffffffffu, at_label);
    mark = (any ? kTaught : 0) | (label >= 0 ? kLabelled | at_label << kSlotShift : 0);
    if (lane == 0) {
      out.slot_id[row * (K + 1) + K] = label >= 0 && at_label == K ? (int)label : -1;
      out.slot_p[row * (K + 1) + K] = 0.f;
      out.info[row] = any ? make_double2(dot * inv_total - log(total), sum_p) : make_double2(0.0, 0.0);
      out.mark[row] = mark;
      if (need) need[row] = mark ? row : -1;
    }
  }
  if (row < rows && lane < kStats) stats[lane * rows + row] = 0.0;
  if (lane == 0) marks[warp] = mark;
  __syncthreads();
  if (threadIdx.x == 0) {
    int2 n = make_int2(0, 0);
    for (int r = 0; r < kPrepareRows; ++r) {
      n.x += (marks[r] & kTaught) != 0;
      n.y += (marks[r] & kLabelled) != 0;
    }
    out.counts[blockIdx.x] = n;
  }
}

// Weights of a row's two gradients, from the number of rows that share them.  `red`: kThreads / 32 values.
struct Weights {
  double taught, labelled;
};
template <int kThreads>
MMT_DEVICE Weights call_weights(const DistillRows& rows, const DistillCall& call, int* red) {
  int t = 0, l = 0;
  for (int i = threadIdx.x; i < rows.n_counts; i += kThreads) {
    const int2 n = rows.counts[i];
    t += n.x;
    l += n.y;
  }
  t = block_total<kThreads>(t, red);
  l = block_total<kThreads>(l, red);
  return {(1.0 - (double)call.share) / max(t, 1), (double)call.share / max(l, 1)};
}

// What a sum of powers below `m` is worth below `top`; nothing for a set of nothing but -inf.
MMT_DEVICE float rescale(float m, float c, float top) { return m == -INFINITY ? 0.f : pow2((m - top) * c); }

// ----------------------------------------------------------------------------
// Statistics of this shard's logits, one CTA per row.  With compacted rows (`src`: the row that each place holds, `cnt`:
// places that are taken) logits go by place, everything else by row.  Shards of a vocabulary come this way, and rows that no
// cluster holds: three passes over memory instead of two.  128 rows of 820008 bf16 (two an SM at most, and few): 153 us, and
// 193 for their gradient, bound by the instructions of a thread's chain.
// ----------------------------------------------------------------------------
template <typename T, bool kDual>
__global__ void __launch_bounds__(kDistillThreads) distill_stats_kernel(const T* logits, long ld, int V, long vocab_lo,
                                                                       DistillRows rows, DistillCall call, long n_rows,
                                                                       const long* src, const int* cnt,
                                                                       double* __restrict__ stats) {
  grid_dependency_sync();
  __shared__ float red[kDistillThreads / 32];
  __shared__ double dred[kDistillThreads / 32];
  if (cnt && (int)blockIdx.x >= *cnt) return;
  const long at = src ? src[blockIdx.x] : (long)blockIdx.x;
  if (at < 0) return;
  const int mark = rows.mark[at];
  if (mark == 0) return;
  const Row<T> row(logits + blockIdx.x * ld, V);
  const int nv = row.vectors();
  float m = -INFINITY, s = 0.f, s1 = 0.f;
  for (int i = threadIdx.x; i < nv; i += kDistillThreads) {
    float v[Row<T>::kVec];
    RowVec<T>::unpack(row.load(i), v);
    float lm = v[0];
#pragma unroll
    for (int j = 1; j < Row<T>::kVec; ++j) lm = fmaxf(lm, v[j]);
    if (lm > m) {
      s *= rescale(m, call.c, lm);
      if (kDual) s1 *= rescale(m, call.c1, lm);
      m = lm;
    }
    // a thread that has seen nothing but -inf adds zeros (2^-inf), not 2^(-inf + inf)
    const float less = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j) {
      s += pow2((v[j] - less) * call.c);
      if (kDual) s1 += pow2((v[j] - less) * call.c1);
    }
  }
  const float gm = block_top<kDistillThreads>(m, red);
  if (gm != -INFINITY) {
    s *= rescale(m, call.c, gm);
    if (kDual) s1 *= rescale(m, call.c1, gm);
  }
  s = block_total<kDistillThreads>(s, red);
  if (kDual) s1 = block_total<kDistillThreads>(s1, red);
  const double zero_at = gm == -INFINITY ? 0.0 : (double)gm;
  double dot = 0.0, mass = 0.0, label = 0.0;
  int mine = 0;
  for (int j = threadIdx.x; j <= rows.K; j += kDistillThreads) {
    const long id = rows.slot_id[at * (rows.K + 1) + j];
    const float p = rows.slot_p[at * (rows.K + 1) + j];
    if (id < 0 || id < vocab_lo || id >= vocab_lo + V) continue;
    const double x = (double)to_float(row.p[id - vocab_lo]) - zero_at;
    if (!(p == 0.f)) dot += (double)p * x * (double)call.c;
    mass += (double)p;
    if ((mark & kLabelled) && j == mark >> kSlotShift) {
      label = x * (double)call.c1;
      mine = 1;
    }
  }
  mine = __syncthreads_or(mine);
  dot = block_total<kDistillThreads>(dot, dred);
  mass = block_total<kDistillThreads>(mass, dred);
  label = block_total<kDistillThreads>(label, dred);
  if (threadIdx.x == 0) {
    stats[kTop * n_rows + at] = (double)gm * (double)call.c;
    stats[kTop1 * n_rows + at] = (double)gm * (double)call.c1;
    stats[kSum * n_rows + at] = s;
    stats[kSum1 * n_rows + at] = kDual ? s1 : s;
    stats[kDot * n_rows + at] = dot;
    stats[kLabel * n_rows + at] = label;
    stats[kMass * n_rows + at] = mass;
    stats[kMine * n_rows + at] = (double)mine;
  }
}

// ----------------------------------------------------------------------------
// Gradient from the whole vocabulary's statistics, one CTA per row, into `out`.
// ----------------------------------------------------------------------------
template <typename T, typename O, bool kDual>
__global__ void __launch_bounds__(kDistillThreads) distill_grad_kernel(const T* logits, long ld, int V, long vocab_lo,
                                                                      DistillRows rows, DistillCall call, long n_rows,
                                                                      const long* src, const int* cnt, const double* stats,
                                                                      const float* dloss, O* out, long out_ld) {
  grid_dependency_sync();
  __shared__ int red[kDistillThreads / 32];
  __shared__ float slot_x[kMaxTop + 1];
  const Row<T> row(logits + blockIdx.x * ld, V);
  O* o = out + blockIdx.x * out_ld;
  const int o_lead = Row<T>::lead_for(o), nv = row.vectors();
  if (cnt) {
    // compacted rows: those behind the last one are not read again, except that the weight gradient's last block of 64
    // rows (the first one if there is none) has to end in zeros
    const int n = *cnt;
    if ((int)blockIdx.x >= n && (int)blockIdx.x >= max((n + 63) / 64 * 64, 64)) return;
  }
  const long at = cnt && (int)blockIdx.x >= *cnt ? -1 : src ? src[blockIdx.x] : (long)blockIdx.x;
  const int mark = at < 0 ? 0 : rows.mark[at];
  if (mark == 0) {
    const float zero[Row<T>::kVec] = {};
    for (int i = threadIdx.x; i < nv; i += kDistillThreads) row.store(o, o_lead, i, zero);
    return;
  }
  const Weights w = call_weights<kDistillThreads>(rows, call, red);
  const float d = dloss ? *dloss : 1.f;
  const float wt = mark & kTaught ? (float)(w.taught * (double)call.temperature) * d : 0.f;
  const float wl = mark & kLabelled ? (float)w.labelled * d : 0.f;
  const float m = (float)(stats[kTop * n_rows + at] / (double)call.c);
  const float a = (kDual ? wt : wt + wl) / (float)stats[kSum * n_rows + at];
  const float a1 = kDual ? wl / (float)stats[kSum1 * n_rows + at] : 0.f;
  for (int j = threadIdx.x; j <= rows.K; j += kDistillThreads) {
    const long id = rows.slot_id[at * (rows.K + 1) + j];
    if (id >= 0 && id >= vocab_lo && id < vocab_lo + V) slot_x[j] = to_float(row.p[id - vocab_lo]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nv; i += kDistillThreads) {
    float v[Row<T>::kVec];
    RowVec<T>::unpack(row.load(i), v);
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j) {
      float g = a * pow2((v[j] - m) * call.c);
      if (kDual) g += a1 * pow2((v[j] - m) * call.c1);
      v[j] = g;
    }
    row.store(o, o_lead, i, v);
  }
  __syncthreads();
  for (int j = threadIdx.x; j <= rows.K; j += kDistillThreads) {
    const long id = rows.slot_id[at * (rows.K + 1) + j];
    if (id < 0 || id < vocab_lo || id >= vocab_lo + V) continue;
    float g = a * pow2((slot_x[j] - m) * call.c);
    if (kDual) g += a1 * pow2((slot_x[j] - m) * call.c1);
    g -= wt * rows.slot_p[at * (rows.K + 1) + j];
    if ((mark & kLabelled) && j == mark >> kSlotShift) g -= wl;
    from_float(g, o + (id - vocab_lo));
  }
}

// ----------------------------------------------------------------------------
// Statistics and gradient of a whole vocabulary in one pass over the logits.  A cluster of C CTAs holds one row in shared
// memory, a run of its vectors each, which a bulk copy brings.  Each CTA reduces its share to (largest, S, S1) and writes
// that into every CTA of the cluster, and behind that exchange all of them know the row's statistics.  A logit is read
// once and its gradient written once.
//
// Second softmax (kMode): none, or that of temperature one for the labels.  If the temperature is two or four, its powers are
// the first one's squared once or twice (c1 = tau c exactly).  A whole step in the case of launch_mode: 193 us with one softmax,
// 202 and 205 with two at temperatures of two and four, 250 at 0.7, 1.5 and 3, where a logit takes two powers.
//
// The parts travel as asynchronous stores that count themselves into an mbarrier of the CTA they go to (two of them, in
// turn: a CTA may be a row ahead of another, never two).  A barrier of the cluster would also wait until the gradients that
// the threads have stored are visible, which is several microseconds.
//
// What bounds it is issue (half of the cycles) and the chain of a row, copy to exchange to gradient, as much as memory (55 %);
// so the rows are visited in an order that mixes neighbours: those without a teacher, which are only cleared, come in long runs
// (image tokens), and their stores run beside the others' arithmetic this way.  The case of launch_mode: 234 us in order, 216
// mixed, both before the second powers' squarings were unrolled; with 256 threads instead of 128, 242 and 232.
//
// Rows are handed out by tickets: a cluster knows its row and the next one, whose copy starts as soon as the row's gradients
// are formed, and takes a ticket for the one after that, which travels with the parts.
// ----------------------------------------------------------------------------
constexpr int kSingle = 0, kTwice = -1;            // or the number of squares
constexpr int kFewThreads = 128;                   // of a CTA that holds a short run

// The two powers of two logits below `m`, with c = (c, c) and so on.
struct Powers {
  f32x2 c, c1, less;
  MMT_DEVICE Powers(const DistillCall& call, float m)
      : c(both(call.c, call.c)), c1(both(call.c1, call.c1)), less(both(-m, -m)) {}
  template <int kMode>
  MMT_DEVICE void take(f32x2 x, f32x2& e, f32x2& e1) const {
    x = add2(x, less);
    float2 v = apart(mul2(x, c));
    e = both(pow2(v.x), pow2(v.y));
    if constexpr (kMode == kTwice) {
      v = apart(mul2(x, c1));
      e1 = both(pow2(v.x), pow2(v.y));
    }
    if constexpr (kMode > 0) {
      e1 = mul2(e, e);
#pragma unroll
      for (int k = 1; k < kMode; ++k) e1 = mul2(e1, e1);
    }
  }
};

template <typename T, typename O, int kThreads, int kMode>
__global__ void __launch_bounds__(kThreads, kThreads == kFewThreads ? 6 : 2)
    distill_fused_kernel(const T* logits, long ld, int V, DistillRows rows, DistillCall call, long n_rows,
                         int places, int step, const long* src, const int* cnt, double* __restrict__ stats,
                         int* ticket, const float* dloss, O* out, long out_ld, int per, MmtErrorWord* ew) {
  grid_dependency_sync();
  constexpr int kVec = Row<T>::kVec, kWarps = kThreads / 32, kFix = (kMaxTop + kThreads) / kThreads;
  constexpr bool kDual = kMode != kSingle;
  extern __shared__ __align__(128) uint4 held[];   // this CTA's vectors of the row, `per` of them
  __shared__ uint64_t arrived, met[2];
  __shared__ int red[kWarps];
  __shared__ float4 warp_part[kWarps];
  __shared__ float4 cta_part[2][kMaxCluster];
  __shared__ int slot_ids[2][kMaxTop + 1];
  __shared__ float slot_ps[2][kMaxTop + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)cluster_size(), rank = (int)cluster_rank(), clusters = gridDim.x / C, first = rank * per;
  if (tid == 0) {
    mbar_init(&arrived, 1);
    mbar_init(&met[0], 1);
    mbar_init(&met[1], 1);
    mbar_fence_init();
  }
  const Weights w = call_weights<kThreads>(rows, call, red);
  const float d = dloss ? *dloss : 1.f;
  const float w_taught = (float)(w.taught * (double)call.temperature) * d, w_labelled = (float)w.labelled * d;
  const double loss_taught = w.taught * (double)call.temperature * (double)call.temperature * kLn2;
  const double loss_labelled = w.labelled * kLn2;
  const int taken = cnt ? *cnt : places;
  // rows behind the last taken one are not read again, except that the weight gradient's last block of 64 rows (the first
  // one if there is none) has to end in zeros
  const int end = cnt ? min(places, max((taken + 63) / 64 * 64, 64)) : places;
  auto row_at = [&](int place) { return place >= taken ? -1 : src ? (int)src[place] : place; };
  auto mark_of = [&](int at) { return at < 0 ? 0 : rows.mark[at]; };
  auto row_of = [&](int place) { return Row<T>(logits + (long)place * ld, V); };
  // Whole vectors of this CTA's run of a row, from the run's first.
  auto whole = [&](const Row<T>& row, int n) {
    const int lo = min(n, (int)(first == 0 && row.lead != 0));
    return make_int2(lo, max(lo, min(n, (row.lead + V) / kVec - first)));
  };
  auto fetch = [&](int place) {
    const Row<T> row = row_of(place);
    const int2 r = whole(row, max(min(per, row.vectors() - first), 0));
    if (r.x >= r.y) return;
    fence_proxy_async_smem();                      // behind what ordinary stores left in `held`
    mbar_expect_tx(&arrived, (r.y - r.x) * 16);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(held + r.x)),
                 "l"(row.p + row.column(first + r.x)), "r"((r.y - r.x) * 16), "r"(smem_u32(&arrived))
                 : "memory");
  };
  cluster_barrier();                               // every CTA has started: its shared memory may be written
  // the q-th row that is handed out
  auto place_of = [&](int q) { return q >= end ? end : step == 1 ? q : (int)((long)q * step % end); };
  int place = place_of(blockIdx.x / C), next = place_of(blockIdx.x / C + clusters);
  int at = place < end ? row_at(place) : -1, mark = mark_of(at);
  if (tid == 0 && mark != 0) fetch(place);
  const int K1 = rows.K + 1;
  // A row's slots on their way into shared memory.
  auto fetch_slots = [&](int at, int turn) {
    for (int j = tid; j < K1; j += kThreads) {
      const long q = (long)at * K1 + j;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&slot_ids[turn][j])), "l"(rows.slot_id + q)
                   : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&slot_ps[turn][j])), "l"(rows.slot_p + q)
                   : "memory");
    }
  };
  if (mark != 0) fetch_slots(at, 0);
  uint32_t phase = 0;
  for (int k = 0; place < end; ++k) {
    const int turn = k & 1;
    int after = 0;
    if (rank == 0 && warp == 0 && lane == 0) after = place_of(2 * clusters + atomicAdd(ticket, 1));
    const Row<T> row = row_of(place);
    const int n = max(min(per, row.vectors() - first), 0);
    const int2 mid = whole(row, n);
    O* o = out ? out + (long)place * out_ld : nullptr;
    const int o_lead = Row<T>::lead_for(o);
    const int next_at = next < end ? row_at(next) : -1, next_mark = mark_of(next_at);
    if (mark != 0) {
      if (tid >= 64 && tid < 64 + n - (mid.y - mid.x)) {
        const int i = tid == 64 && mid.x ? 0 : n - 1;
        held[i] = row.load(first + i);
      }
      // one warp waits for the copy, the others without issuing anything at the barrier
      if (mid.x < mid.y) {
        if (warp == 0) mbar_wait(&arrived, phase, ew, 710);
        phase ^= 1;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();
      float m = -INFINITY;
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads) m = thread_max(held[i], m, T());
      m = warp_top(m);
      // a warp that has nothing but -inf adds zeros (2^-inf), not 2^(-inf + inf)
      f32x2 s2 = both(0.f, 0.f), s12 = s2;
      {
        const Powers pw(call, m == -INFINITY ? 0.f : m);
#pragma unroll 2
        for (int i = tid; i < n; i += kThreads) {
          float v[kVec];
          RowVec<T>::unpack(held[i], v);
#pragma unroll
          for (int j = 0; j < kVec; j += 2) {
            f32x2 e, e1;
            pw.take<kMode>(both(v[j], v[j + 1]), e, e1);
            s2 = add2(s2, e);
            if constexpr (kDual) s12 = add2(s12, e1);
          }
        }
      }
      float s = warp_sum(apart(s2).x + apart(s2).y), s1 = apart(s12).x + apart(s12).y;
      if constexpr (kDual) s1 = warp_sum(s1);
      if (lane == 0) warp_part[warp] = make_float4(m, s, s1, 0.f);
      __syncthreads();
    }
    if (warp == 0) {
      after = __shfl_sync(0xffffffffu, after, 0);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      if (mark != 0) {
        a = warp_part[lane % kWarps];
        const float top = warp_top(a.x);
        a.y *= rescale(a.x, call.c, top);
        if constexpr (kDual) a.z *= rescale(a.x, call.c1, top);
        a.x = top;
#pragma unroll
        for (int q = kWarps / 2; q > 0; q >>= 1) {
          a.y += __shfl_xor_sync(0xffffffffu, a.y, q);
          if constexpr (kDual) a.z += __shfl_xor_sync(0xffffffffu, a.z, q);
        }
      }
      a.w = __int_as_float(after);
      if (lane == 0) mbar_expect_tx(&met[turn], C * 16);
      __syncwarp();
      if (lane < C) cluster_send(&cta_part[turn][rank], &met[turn], lane, a);
    }
    if (mark == 0 && o) {
      const float zero[kVec] = {};
      for (int i = tid; i < n; i += kThreads) row.store(o, o_lead, first + i, zero);
    }
    if (warp == 0) cluster_wait(&met[turn], k >> 1 & 1, ew, 711);
    __syncthreads();
    after = __float_as_int(cta_part[turn][0].w);
    if (mark != 0) {
      // lane q of every warp takes CTA q's part
      const float4 part = cta_part[turn][lane % C];
      const float top = warp_top(part.x);
      float S = part.y * rescale(part.x, call.c, top), S1 = kDual ? part.z * rescale(part.x, call.c1, top) : 0.f;
      for (int q = C / 2; q > 0; q >>= 1) {
        S += __shfl_xor_sync(0xffffffffu, S, q);
        if constexpr (kDual) S1 += __shfl_xor_sync(0xffffffffu, S1, q);
      }
      const int label_at = mark & kLabelled ? mark >> kSlotShift : -1;
      const float wt = mark & kTaught ? w_taught : 0.f, wl = mark & kLabelled ? w_labelled : 0.f;
      const float a = (kDual ? wt : wt + wl) / S, a1 = kDual ? wl / S1 : 0.f;
      const Powers pw(call, top);
      const f32x2 a2 = both(a, a), a12 = both(a1, a1);
      auto grad = [&](float x, float y) {
        f32x2 e, e1;
        pw.take<kMode>(both(x, y), e, e1);
        return apart(kDual ? fma2(a2, e, mul2(a12, e1)) : mul2(a2, e));
      };
      auto grads = [&](int i, float (&v)[kVec]) {
        RowVec<T>::unpack(held[i], v);
#pragma unroll
        for (int j = 0; j < kVec; j += 2) {
          const float2 g = grad(v[j], v[j + 1]);
          v[j] = g.x;
          v[j + 1] = g.y;
        }
      };
      if (o) {
        const bool in_step = o_lead == row.lead;   // whole vectors may be stored whole
        const int lo = in_step ? mid.x : 0, hi = in_step ? mid.y : n;
#pragma unroll 2
        for (int i = lo + tid; i < hi; i += kThreads) {
          float v[kVec];
          grads(i, v);
          if (in_step) Row<T>::store_whole(o + row.column(first + i), v);
          else row.store(o, o_lead, first + i, v);
        }
        if (tid >= kThreads - n + (hi - lo)) {     // the others
          const int i = tid == kThreads - 1 && lo ? 0 : n - 1;
          float v[kVec];
          grads(i, v);
          row.store(o, o_lead, first + i, v);
        }
      }
      // the slots that this CTA holds: their gradients (kFix slots a thread at most), and one warp's part of the row's loss
      auto held_slot = [&](int j, int& id, float& p, float& x) {
        id = j < K1 ? slot_ids[turn][j] : -1;
        if (id < 0 || (unsigned)((id + row.lead) / kVec - first) >= (unsigned)n) return false;
        p = slot_ps[turn][j];
        x = to_float(reinterpret_cast<const T*>(held)[id + row.lead - first * kVec]);
        return true;
      };
      int id;
      float p, x, fix[kFix];
      int fix_at[kFix];
#pragma unroll
      for (int b = 0; b < kFix; ++b) {
        const int j = tid + b * kThreads;
        fix_at[b] = -1;
        if (!held_slot(j, id, p, x)) continue;
        fix_at[b] = id;
        fix[b] = grad(x, x).x - wt * p - (j == label_at ? wl : 0.f);
      }
      double part_loss = 0.0;
      if (warp == kWarps - 1) {
        const double lse = log2((double)S), lse1 = kDual ? log2((double)S1) : lse;         // above m c
        for (int j = lane; j < K1; j += 32)
          if (held_slot(j, id, p, x)) {
            if (!(p == 0.f)) part_loss += loss_taught * (double)p * (lse - ((double)x - (double)top) * (double)call.c);
            if (j == label_at) part_loss += loss_labelled * (lse1 - ((double)x - (double)top) * (double)call.c1);
          }
      }
      __syncthreads();                             // `held` may be written again; a slot's gradient was another thread's
      if (tid == 0 && next_mark != 0) fetch(next);
      if (o) {
#pragma unroll
        for (int b = 0; b < kFix; ++b)
          if (fix_at[b] >= 0) from_float(fix[b], o + fix_at[b]);
      }
      if (warp == kWarps - 1) {
#pragma unroll
        for (int q = 16; q > 0; q >>= 1) part_loss += __shfl_xor_sync(0xffffffffu, part_loss, q);
        if (lane == 0) {
          if (rank == 0 && (mark & kTaught) && loss_taught > 0.0) part_loss += loss_taught / kLn2 * rows.info[at].x;
          stats[(long)rank * n_rows + at] = part_loss;
        }
      }
    } else {
      __syncthreads();                             // all have read the ticket
      if (tid == 0 && next_mark != 0) fetch(next);
    }
    if (next_mark != 0) fetch_slots(next_at, turn ^ 1);
    place = next;
    next = after;
    at = next_at;
    mark = next_mark;
  }
  // the last cluster puts the tickets back for the next launch
  if (rank == 0 && tid == 0 && atomicAdd(ticket + 1, 1) == clusters - 1) ticket[0] = ticket[1] = 0;
}

// ----------------------------------------------------------------------------
// Losses of the rows from their statistics.
// ----------------------------------------------------------------------------
__global__ void __launch_bounds__(256) distill_row_loss_kernel(DistillRows rows, DistillCall call, long n_rows,
                                                               double* stats) {
  grid_dependency_sync();
  __shared__ int red[8];
  const Weights w = call_weights<256>(rows, call, red);
  const long r = blockIdx.x * 256L + threadIdx.x;
  if (r >= n_rows) return;
  const int mark = rows.mark[r];
  double loss = 0.0;
  if ((mark & kTaught) && w.taught > 0.0) {
    const double2 info = rows.info[r];
    const double kl = info.x - kLn2 * (stats[kDot * n_rows + r] - info.y * log2(stats[kSum * n_rows + r]));
    loss += w.taught * (double)call.temperature * (double)call.temperature * kl;
  }
  if ((mark & kLabelled) && w.labelled > 0.0)
    loss += w.labelled * kLn2 * (log2(stats[kSum1 * n_rows + r]) - stats[kLabel * n_rows + r]);
  stats[kLoss * n_rows + r] = loss;
}

// The sum of n losses, always in the same order: one CTA, 4 us for 2048 rows of 8 parts.
constexpr int kLossThreads = 1024;
__global__ void __launch_bounds__(kLossThreads) distill_loss_kernel(const double* losses, long n, float* __restrict__ loss) {
  grid_dependency_sync();
  __shared__ double dred[kLossThreads / 32];
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  long i = threadIdx.x;
  for (; i + 3 * kLossThreads < n; i += 4 * kLossThreads)
#pragma unroll
    for (int q = 0; q < 4; ++q) part[q] += losses[i + q * kLossThreads];
  for (; i < n; i += kLossThreads) part[0] += losses[i];
  double total = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((threadIdx.x & 31) == 0) dred[threadIdx.x >> 5] = total;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  total = dred[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (threadIdx.x == 0) *loss = (float)total;
}

// grad *= *factor, unless that is one, which is seen in 3 us without a pass over memory.
template <typename T>
__global__ void __launch_bounds__(256) distill_scale_kernel(T* grad, long n, const float* factor) {
  grid_dependency_sync();
  const float f = *factor;
  if (f == 1.f) return;
  constexpr int kVec = Row<T>::kVec;
  const long step = (long)gridDim.x * blockDim.x, first = blockIdx.x * (long)blockDim.x + threadIdx.x;
  for (long i = first; i < n / kVec; i += step) {
    float v[kVec];
    RowVec<T>::unpack(*reinterpret_cast<const uint4*>(grad + i * kVec), v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] *= f;
    *reinterpret_cast<uint4*>(grad + i * kVec) = RowVec<T>::pack(v);
  }
  const long e = n / kVec * kVec + first;
  if (e < n) from_float(to_float(grad[e]) * f, grad + e);
}

// out[r] = sum over the runs of parts[run][r], in their order, for the first min(*cnt, rows) rows of `cols` (a multiple of 8):
// what mmt_gemm_bf16_split leaves.  13 runs of 256 x 2048, still in L2: 9 us.
__global__ void __launch_bounds__(256) sum_runs_kernel(const float* parts, int runs, const int* cnt, int rows, int cols,
                                                       bf16* __restrict__ out) {
  grid_dependency_sync();
  const long n8 = (long)min(max(*cnt, 0), rows) * cols / 8, stride = (long)rows * cols;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n8; i += gridDim.x * 256L) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int r = 0; r < runs; ++r) {
      const float4* p = reinterpret_cast<const float4*>(parts + r * stride + i * 8);
      const float4 x = p[0], y = p[1];
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
    }
    *reinterpret_cast<uint4*>(out + i * 8) =
        make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
  }
}

}  // namespace

// The words of a call, in the order of ops/vocab_rows.py.
struct MmtDistill {
  const void* logits;
  void* out;
  long ld, out_ld, vocab_lo;
  long rows;                        // of the batch
  long places;                      // rows of `logits`
  const long* src;                  // compacted rows, or null
  const int* cnt;
  int* slot_id;
  float* slot_p;
  double* info;
  int* mark;
  int* counts;
  double* stats;
  int* ticket;                      // two words, zero between launches
  const float* dloss;
  double temperature, share;
  int V, K, is_f32, out_f32;
  int parts;                        // of a row's loss in `stats`, 0: its statistics; set by the kernels' calls
};

namespace {

constexpr double kLog2e = 1.44269504088896340736;

DistillRows rows_of(const MmtDistill& d) {
  return {d.slot_id, d.slot_p, reinterpret_cast<double2*>(d.info), d.mark, reinterpret_cast<int2*>(d.counts), d.K,
          (int)((d.rows + kPrepareRows - 1) / kPrepareRows)};
}
DistillCall call_of(const MmtDistill& d) {
  return {(float)(kLog2e / d.temperature), (float)kLog2e, (float)d.temperature, (float)d.share};
}
bool dual(const MmtDistill& d) { return d.share > 0.0 && d.temperature != 1.0; }
constexpr long kMostRows = 0x7fff0000L;            // tickets are a few thousand more, and ints
bool wrong(const MmtDistill& d) {
  return d.K < 1 || d.K > kMaxTop || d.V < 1 || d.rows < 0 || d.places < 0 || d.rows > kMostRows || d.places > kMostRows;
}

template <typename T, bool kDual>
int launch_stats(const MmtDistill& d, void* stream) {
  return (int)launch_dependent(distill_stats_kernel<T, kDual>, (unsigned)d.places, kDistillThreads, 0, VR_STREAM(stream),
                               reinterpret_cast<const T*>(d.logits), d.ld, d.V, d.vocab_lo, rows_of(d), call_of(d), d.rows,
                               d.src, d.cnt, d.stats);
}
template <typename T, typename O, bool kDual>
int launch_grad(const MmtDistill& d, void* stream) {
  return (int)launch_dependent(distill_grad_kernel<T, O, kDual>, (unsigned)d.places, kDistillThreads, 0, VR_STREAM(stream),
                               reinterpret_cast<const T*>(d.logits), d.ld, d.V, d.vocab_lo, rows_of(d), call_of(d), d.rows,
                               d.src, d.cnt, d.stats, d.dloss, reinterpret_cast<O*>(d.out), d.out_ld);
}

// Vectors that a row has at most, wherever it starts.
long row_vectors(const MmtDistill& d) {
  const int vec = d.is_f32 ? 4 : 8;
  return (d.V + vec - 2) / vec + 1;
}

// A step through n rows that visits them all, each far from the one before.
int mixing_step(int n) {
  int s = (int)(0.618 * n);
  while (s > 1 && std::gcd(s, n) != 1) --s;
  return s < 1 ? 1 : s;
}

constexpr int kHeldBytes = 39 * 1024, kMaxHeldBytes = 200 * 1024;

template <typename T, typename O, int kThreads, int kMode>
int launch_held(MmtDistill& d, int C, int per, void* stream) {
  d.parts = max(d.parts, C);                // chunks of a batch differ in it
  auto kernel = distill_fused_kernel<T, O, kThreads, kMode>;
  static int allowed = 0;
  const int bytes = per * 16;
  if (bytes > allowed) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxHeldBytes);
    if (e != cudaSuccess) return (int)e;
    allowed = kMaxHeldBytes;
  }
  thread_local int known_C = 0, known_bytes = 0, most = 0;
  if (C != known_C || bytes != known_bytes) {
    most = resident_clusters(kernel, kThreads, C, bytes);
    known_C = C;
    known_bytes = bytes;
  }
  const long clusters = d.places < most ? d.places : most;
  const int step = d.cnt ? 1 : mixing_step((int)d.places);
  return (int)launch_cluster(kernel, (unsigned)(clusters * C), kThreads, C, bytes, VR_STREAM(stream),
                             reinterpret_cast<const T*>(d.logits), d.ld, d.V, rows_of(d), call_of(d), d.rows,
                             (int)d.places, step, d.src, d.cnt, d.stats, d.ticket, d.dloss, reinterpret_cast<O*>(d.out),
                             d.out_ld, per, mmt_error_word());
}
template <typename T, typename O, int kMode>
int launch_mode(MmtDistill& d, void* stream) {
  const long nv = row_vectors(d);
  // As few CTAs a row as hold it in 39 KB each, of which an SM has five (smaller runs: six); more where there are few rows.
  // 2048 x 152064 bf16, half of the rows with a teacher, two softmaxes at a temperature of two: 200 us in runs of 37 KB, 215 in
  // runs of 75 KB with two CTAs an SM.  512 x 152064 fp32, which eight CTAs hold in 75 KB each: 108 us with 256 threads, 110
  // with 512.
  int C = 1;
  while (C < kMaxCluster && nv * 16 > (long)kHeldBytes * C) C *= 2;
  while (C < kMaxCluster && d.places * C * 2 <= 2 * mmt_sm_count() && nv > 512L * C) C *= 2;
  const int per = (int)((nv + C - 1) / C);
  return per * 16 <= kHeldBytes ? launch_held<T, O, kFewThreads, kMode>(d, C, per, stream)
                                : launch_held<T, O, 256, kMode>(d, C, per, stream);
}
template <typename T, typename O>
int launch_fused(MmtDistill& d, void* stream) {
  if (!dual(d)) return launch_mode<T, O, kSingle>(d, stream);
  if (d.temperature == 2.0) return launch_mode<T, O, 1>(d, stream);
  if (d.temperature == 4.0) return launch_mode<T, O, 2>(d, stream);
  return launch_mode<T, O, kTwice>(d, stream);
}

}  // namespace

extern "C" {

// Size of MmtDistill, for the caller to agree on.
int mmt_distill_bytes() { return (int)sizeof(MmtDistill); }
// Values that `stats` has per row.
int mmt_distill_stats_count() { return kStats; }
// Rows that share one entry of `counts`.
int mmt_distill_count_rows() { return kPrepareRows; }

// Teacher's side of `rows` rows: ids [rows, K] and logits [rows, K] (bf16 or fp32), labels [rows] or null.
// need [rows] or null: the row itself if it has a teacher or a label, -1 for one without.
int mmt_distill_prepare(const MmtDistill* d, const long* ids, long ids_ld, const void* teacher, long teacher_ld,
                        int teacher_f32, const long* labels, long vocab, long* need, void* stream) {
  if (wrong(*d) || vocab > 0x7fffffffL) return -2;
  if (d->rows == 0) return 0;
  const unsigned grid = (unsigned)((d->rows + kPrepareRows - 1) / kPrepareRows);
  const double inv = 1.0 / d->temperature;
  if (teacher_f32)
    return (int)launch_dependent(distill_prepare_kernel<float>, grid, 32 * kPrepareRows, 0, VR_STREAM(stream), ids, ids_ld,
                                 reinterpret_cast<const float*>(teacher), teacher_ld, labels, d->rows, vocab, inv,
                                 (int)(d->share < 1.0), rows_of(*d), need, d->stats, d->ticket, mmt_error_word());
  return (int)launch_dependent(distill_prepare_kernel<bf16>, grid, 32 * kPrepareRows, 0, VR_STREAM(stream), ids, ids_ld,
                               reinterpret_cast<const bf16*>(teacher), teacher_ld, labels, d->rows, vocab, inv,
                               (int)(d->share < 1.0), rows_of(*d), need, d->stats, d->ticket, mmt_error_word());
}

int mmt_distill_stats(MmtDistill* d, void* stream) {
  if (wrong(*d)) return -2;
  d->parts = 0;
  if (d->places == 0) return 0;
  if (d->is_f32) return dual(*d) ? launch_stats<float, true>(*d, stream) : launch_stats<float, false>(*d, stream);
  return dual(*d) ? launch_stats<bf16, true>(*d, stream) : launch_stats<bf16, false>(*d, stream);
}

int mmt_distill_grad(const MmtDistill* d, void* stream) {
  if (wrong(*d) || (d->out_f32 && !d->is_f32)) return -2;
  if (d->places == 0) return 0;
  if (d->out_f32) return dual(*d) ? launch_grad<float, float, true>(*d, stream) : launch_grad<float, float, false>(*d, stream);
  if (d->is_f32) return dual(*d) ? launch_grad<float, bf16, true>(*d, stream) : launch_grad<float, bf16, false>(*d, stream);
  return dual(*d) ? launch_grad<bf16, bf16, true>(*d, stream) : launch_grad<bf16, bf16, false>(*d, stream);
}

// Most columns that mmt_distill_fused takes.
long mmt_distill_fused_columns(int is_f32) {
  return ((long)kMaxHeldBytes / 16 * kMaxCluster - 1) * (is_f32 ? 4 : 8);
}

// Statistics of a whole vocabulary and, unless `out` is null, the gradient (times *dloss, if that is not null).
int mmt_distill_fused(MmtDistill* d, void* stream) {
  if (wrong(*d) || (d->out_f32 && !d->is_f32) || d->V > mmt_distill_fused_columns(d->is_f32)) return -2;
  if (d->places == 0) return 0;
  if (d->out_f32) return launch_fused<float, float>(*d, stream);
  return d->is_f32 ? launch_fused<float, bf16>(*d, stream) : launch_fused<bf16, bf16>(*d, stream);
}

// From the statistics (parts == 0) or from the losses that mmt_distill_fused has left: `parts` for each row.
int mmt_distill_loss(const MmtDistill* d, float* loss, void* stream) {
  if (wrong(*d) || d->parts < 0 || d->parts > kMaxCluster) return -2;
  if (d->parts == 0 && d->rows > 0) {
    const int e = (int)launch_dependent(distill_row_loss_kernel, (unsigned)((d->rows + 255) / 256), 256, 0, VR_STREAM(stream),
                                        rows_of(*d), call_of(*d), d->rows, d->stats);
    if (e) return e;
  }
  return (int)launch_dependent(distill_loss_kernel, 1, kLossThreads, 0, VR_STREAM(stream),
                               d->parts ? d->stats : d->stats + kLoss * d->rows, d->rows * (d->parts ? d->parts : 1), loss);
}

// The sum of the runs of a product whose K was cut (mmt_gemm_bf16_split), as [rows, cols] bf16.
int mmt_sum_runs(const float* parts, int runs, const int* cnt, int rows, int cols, void* out, void* stream) {
  if (cols % 8 || runs < 1) return -2;
  if (rows == 0 || cols == 0) return 0;
  const long want = ((long)rows * cols / 8 + 255) / 256, most = 8L * mmt_sm_count();
  return (int)launch_dependent(sum_runs_kernel, (unsigned)(want < most ? want : most), 256, 0, VR_STREAM(stream), parts, runs,
                               cnt, rows, cols, reinterpret_cast<bf16*>(out));
}

// n values at a 16-byte boundary.
int mmt_distill_scale(void* grad, int is_f32, long n, const float* factor, void* stream) {
  if (n == 0) return 0;
  const long vecs = (n + 7) / 8, want = (vecs + 255) / 256, most = 4L * mmt_sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  return is_f32 ? (int)launch_dependent(distill_scale_kernel<float>, grid, 256, 0, VR_STREAM(stream),
                                        reinterpret_cast<float*>(grad), n, factor)
                : (int)launch_dependent(distill_scale_kernel<bf16>, grid, 256, 0, VR_STREAM(stream),
                                        reinterpret_cast<bf16*>(grad), n, factor);
}

}  // extern "C"
