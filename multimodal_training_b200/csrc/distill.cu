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
// Powers of two: with c = log2(e) / tau rounded to fp32, q_v = 2^(x_v c - top) / S, top = fl(max x * c), S = sum 2^(x c - top).
// Statistics and gradient use the same rounded c and top, so their rounding changes the temperature by 2^-24 and
// nothing else.  S is summed in fp32 (relative error of a few 2^-24); everything that is K long is fp64.
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

// Per row, in statistics of [6][rows]: top and top1 = fl(max x * c1), S and S1, sum of p x over the slots of this shard,
// the label's logit if it is in this shard.
enum { kTop, kTop1, kSum, kSum1, kDot, kLabel, kStats };

// ----------------------------------------------------------------------------
// Teacher's side: one warp per row.  An entry is absent if its id is negative or its logit -inf.
// ----------------------------------------------------------------------------
constexpr int kPrepareWarps = 8, kPrepareRows = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kPrepareWarps) distill_prepare_kernel(const long* ids, long ids_ld, const T* teacher,
                                                                            long teacher_ld, const long* labels, long rows,
                                                                            long vocab, double inv_temperature,
                                                                            DistillRows out, long* need,
                                                                            MmtErrorWord* ew) {
  grid_dependency_sync();
  __shared__ int s_id[kPrepareWarps][kMaxTop];
  __shared__ double s_p[kPrepareWarps][kMaxTop];
  __shared__ int n_taught, n_labelled;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = out.K;
  if (threadIdx.x == 0) n_taught = n_labelled = 0;
  __syncthreads();
  for (int r = warp; r < kPrepareRows; r += kPrepareWarps) {
    const long row = (long)blockIdx.x * kPrepareRows + r;
    if (row >= rows) break;
    double top = -INFINITY;
    bool any = false, odd = false;                  // odd: a logit that is not a number
    for (int j = lane; j < K; j += 32) {
      long id = ids[row * ids_ld + j];
      if (id >= vocab) {
        mmt_report(ew, MMT_ERR_BOUNDS, 700, (int)row);
        id = -1;
      }
      const float t = to_float(teacher[row * teacher_ld + j]);
      const bool here = id >= 0 && !(t == -INFINITY);
      s_id[warp][j] = here ? (int)id : -1;
      s_p[warp][j] = here ? (double)t * inv_temperature : -INFINITY;
      any |= here;
      odd |= here && !(t == t);
      if (here) top = fmax(top, (double)t * inv_temperature);
    }
    any = __any_sync(0xffffffffu, any);
    odd = __any_sync(0xffffffffu, odd);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (odd) top = NAN;
    double total = 0.0, dot = 0.0;
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
    __syncwarp();
    long label = labels ? labels[row] : -1;
    if (label >= vocab) {
      if (lane == 0) mmt_report(ew, MMT_ERR_BOUNDS, 701, (int)row);
      label = -1;
    }
    // an id that the teacher gives more than once has the sum of its probabilities, in the first of its slots
    double sum_p = 0.0;
    int at_label = K;
    for (int j = lane; j < K; j += 32) {
      const int id = s_id[warp][j];
      bool first = id >= 0;
      double p = 0.0;
      if (first) {
        for (int i = 0; i < j; ++i) first &= s_id[warp][i] != id;
        if (first)
          for (int i = j; i < K; ++i) p += s_id[warp][i] == id ? s_p[warp][i] : 0.0;
      }
      const float rounded = first ? (float)(p / total) : 0.f;
      out.slot_id[row * (K + 1) + j] = first ? id : -1;
      out.slot_p[row * (K + 1) + j] = rounded;
      sum_p += (double)rounded;
      if (first && id == label) at_label = j;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum_p += __shfl_xor_sync(0xffffffffu, sum_p, o);
      at_label = min(at_label, __shfl_xor_sync(0xffffffffu, at_label, o));
    }
    if (lane == 0) {
      out.slot_id[row * (K + 1) + K] = label >= 0 && at_label == K ? (int)label : -1;
      out.slot_p[row * (K + 1) + K] = 0.f;
      out.info[row] = any ? make_double2(dot / total - log(total), sum_p) : make_double2(0.0, 0.0);
      out.mark[row] = (any ? kTaught : 0) | (label >= 0 ? kLabelled | at_label << kSlotShift : 0);
      if (need) need[row] = any || label >= 0 ? 0 : -1;
      if (any) atomicAdd(&n_taught, 1);
      if (label >= 0) atomicAdd(&n_labelled, 1);
    }
    __syncwarp();
  }
  __syncthreads();
  if (threadIdx.x == 0) out.counts[blockIdx.x] = make_int2(n_taught, n_labelled);
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

// ----------------------------------------------------------------------------
// Statistics of this shard's logits, one CTA per row.  With compacted rows (`src`: the row that each place holds, `cnt`:
// places that are taken) logits go by place, everything else by row.
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
  if (mark == 0) {
    if (threadIdx.x < kStats) stats[threadIdx.x * n_rows + at] = threadIdx.x == kSum || threadIdx.x == kSum1 ? 1.0 : 0.0;
    return;
  }
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
      s *= exp2f(__fmul_rn(m, call.c) - __fmul_rn(lm, call.c));
      if (kDual) s1 *= exp2f(__fmul_rn(m, call.c1) - __fmul_rn(lm, call.c1));
      m = lm;
    }
    // a thread that has seen nothing but -inf adds zeros (2^-inf), not 2^(-inf + inf)
    const float t = m == -INFINITY ? 0.f : __fmul_rn(m, call.c), t1 = m == -INFINITY ? 0.f : __fmul_rn(m, call.c1);
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j) {
      s += exp2f(__fmaf_rn(v[j], call.c, -t));
      if (kDual) s1 += exp2f(__fmaf_rn(v[j], call.c1, -t1));
    }
  }
  const float gm = block_top<kDistillThreads>(m, red);
  const float t = __fmul_rn(gm, call.c), t1 = __fmul_rn(gm, call.c1);
  if (gm != -INFINITY) {                                       // 0 * 2^-inf for a thread without a logit
    s *= exp2f(__fmul_rn(m, call.c) - t);
    if (kDual) s1 *= exp2f(__fmul_rn(m, call.c1) - t1);
  }
  s = block_total<kDistillThreads>(s, red);
  if (kDual) s1 = block_total<kDistillThreads>(s1, red);
  double dot = 0.0, label = 0.0;
  for (int j = threadIdx.x; j <= rows.K; j += kDistillThreads) {
    const long id = rows.slot_id[at * (rows.K + 1) + j];
    const float p = rows.slot_p[at * (rows.K + 1) + j];
    if (id < 0 || id < vocab_lo || id >= vocab_lo + V) continue;
    const float x = to_float(row.p[id - vocab_lo]);
    if (!(p == 0.f)) dot += (double)p * (double)x;
    if ((mark & kLabelled) && j == mark >> kSlotShift) label = (double)x;
  }
  dot = block_total<kDistillThreads>(dot, dred);
  label = block_total<kDistillThreads>(label, dred);
  if (threadIdx.x == 0) {
    stats[kTop * n_rows + at] = t;
    stats[kTop1 * n_rows + at] = t1;
    stats[kSum * n_rows + at] = s;
    stats[kSum1 * n_rows + at] = kDual ? s1 : s;
    stats[kDot * n_rows + at] = dot;
    stats[kLabel * n_rows + at] = label;
  }
}

// ----------------------------------------------------------------------------
// Gradient from the whole vocabulary's statistics, one CTA per row, into `out` (which may be the logits).
// ----------------------------------------------------------------------------
template <typename T, bool kDual>
__global__ void __launch_bounds__(kDistillThreads) distill_grad_kernel(const T* logits, long ld, int V, long vocab_lo,
                                                                      DistillRows rows, DistillCall call, long n_rows,
                                                                      const long* src, const int* cnt, const double* stats,
                                                                      const float* dloss, T* out, long out_ld) {
  grid_dependency_sync();
  __shared__ int red[kDistillThreads / 32];
  __shared__ float slot_x[kMaxTop + 1];
  const Row<T> row(logits + blockIdx.x * ld, V);
  T* o = out + blockIdx.x * out_ld;
  const int o_lead = Row<T>::lead_of(o), nv = row.vectors();
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
  const float t = (float)stats[kTop * n_rows + at], t1 = (float)stats[kTop1 * n_rows + at];
  const float a = (kDual ? wt : wt + wl) / (float)stats[kSum * n_rows + at];
  const float a1 = kDual ? wl / (float)stats[kSum1 * n_rows + at] : 0.f;
  for (int j = threadIdx.x; j <= rows.K; j += kDistillThreads) {
    const long id = rows.slot_id[at * (rows.K + 1) + j];
    if (id >= 0 && id >= vocab_lo && id < vocab_lo + V) slot_x[j] = to_float(row.p[id - vocab_lo]);
  }
  __syncthreads();                                            // the logits are written over below
  for (int i = threadIdx.x; i < nv; i += kDistillThreads) {
    float v[Row<T>::kVec];
    RowVec<T>::unpack(row.load(i), v);
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j) {
      float g = a * exp2f(__fmaf_rn(v[j], call.c, -t));
      if (kDual) g += a1 * exp2f(__fmaf_rn(v[j], call.c1, -t1));
      v[j] = g;
    }
    row.store(o, o_lead, i, v);
  }
  __syncthreads();
  for (int j = threadIdx.x; j <= rows.K; j += kDistillThreads) {
    const long id = rows.slot_id[at * (rows.K + 1) + j];
    if (id < 0 || id < vocab_lo || id >= vocab_lo + V) continue;
    float g = a * exp2f(__fmaf_rn(slot_x[j], call.c, -t));
    if (kDual) g += a1 * exp2f(__fmaf_rn(slot_x[j], call.c1, -t1));
    g -= wt * rows.slot_p[at * (rows.K + 1) + j];
    if ((mark & kLabelled) && j == mark >> kSlotShift) g -= wl;
    from_float(g, o + (id - vocab_lo));
  }
}

// ----------------------------------------------------------------------------
// The loss of all rows, in the order of the rows: one CTA.
// ----------------------------------------------------------------------------
constexpr int kLossThreads = 1024;
__global__ void __launch_bounds__(kLossThreads) distill_loss_kernel(DistillRows rows, DistillCall call, long n_rows,
                                                                   const double* stats, float* __restrict__ loss) {
  grid_dependency_sync();
  __shared__ double dred[kLossThreads / 32];
  __shared__ int red[kLossThreads / 32];
  const Weights w = call_weights<kLossThreads>(rows, call, red);
  double total = 0.0;
  for (long r = threadIdx.x; r < n_rows; r += kLossThreads) {
    const int mark = rows.mark[r];
    if ((mark & kTaught) && w.taught > 0.0) {
      const double2 info = rows.info[r];
      const double lse = stats[kTop * n_rows + r] + log2(stats[kSum * n_rows + r]);
      const double kl = info.x - kLn2 * (stats[kDot * n_rows + r] * (double)call.c - info.y * lse);
      total += w.taught * (double)call.temperature * (double)call.temperature * kl;
    }
    if ((mark & kLabelled) && w.labelled > 0.0) {
      const double lse = stats[kTop1 * n_rows + r] + log2(stats[kSum1 * n_rows + r]);
      total += w.labelled * kLn2 * (lse - stats[kLabel * n_rows + r] * (double)call.c1);
    }
  }
  total = block_total<kLossThreads>(total, dred);
  if (threadIdx.x == 0) *loss = (float)total;
}

// grad *= *factor, unless that is one.
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
  const float* dloss;
  double temperature, share;
  int V, K, is_f32;
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
bool wrong(const MmtDistill& d) {
  return d.K < 1 || d.K > kMaxTop || d.V < 1 || d.rows < 0 || d.places < 0 || d.places > 0x7fffffffL;
}

template <typename T, bool kDual>
int launch_stats(const MmtDistill& d, void* stream) {
  return (int)launch_dependent(distill_stats_kernel<T, kDual>, (unsigned)d.places, kDistillThreads, 0, VR_STREAM(stream),
                               reinterpret_cast<const T*>(d.logits), d.ld, d.V, d.vocab_lo, rows_of(d), call_of(d), d.rows,
                               d.src, d.cnt, d.stats);
}
template <typename T, bool kDual>
int launch_grad(const MmtDistill& d, void* stream) {
  return (int)launch_dependent(distill_grad_kernel<T, kDual>, (unsigned)d.places, kDistillThreads, 0, VR_STREAM(stream),
                               reinterpret_cast<const T*>(d.logits), d.ld, d.V, d.vocab_lo, rows_of(d), call_of(d), d.rows,
                               d.src, d.cnt, d.stats, d.dloss, reinterpret_cast<T*>(d.out), d.out_ld);
}

}  // namespace

extern "C" {

// Size of MmtDistill, for the caller to agree on.
int mmt_distill_bytes() { return (int)sizeof(MmtDistill); }
// Rows that share one entry of `counts`.
int mmt_distill_count_rows() { return kPrepareRows; }

// Teacher's side of `rows` rows: ids [rows, K] and logits [rows, K] (bf16 or fp32), labels [rows] or null.
// need [rows] or null: 0 for a row with a teacher or a label, -1 for one without.
int mmt_distill_prepare(const MmtDistill* d, const long* ids, long ids_ld, const void* teacher, long teacher_ld,
                        int teacher_f32, const long* labels, long vocab, long* need, void* stream) {
  if (wrong(*d) || vocab > 0x7fffffffL) return -2;
  if (d->rows == 0) return 0;
  const unsigned grid = (unsigned)((d->rows + kPrepareRows - 1) / kPrepareRows);
  const double inv = 1.0 / d->temperature;
  if (teacher_f32)
    return (int)launch_dependent(distill_prepare_kernel<float>, grid, 32 * kPrepareWarps, 0, VR_STREAM(stream), ids, ids_ld,
                                 reinterpret_cast<const float*>(teacher), teacher_ld, labels, d->rows, vocab, inv,
                                 rows_of(*d), need, mmt_error_word());
  return (int)launch_dependent(distill_prepare_kernel<bf16>, grid, 32 * kPrepareWarps, 0, VR_STREAM(stream), ids, ids_ld,
                               reinterpret_cast<const bf16*>(teacher), teacher_ld, labels, d->rows, vocab, inv, rows_of(*d),
                               need, mmt_error_word());
}

int mmt_distill_stats(const MmtDistill* d, void* stream) {
  if (wrong(*d)) return -2;
  if (d->places == 0) return 0;
  if (d->is_f32) return dual(*d) ? launch_stats<float, true>(*d, stream) : launch_stats<float, false>(*d, stream);
  return dual(*d) ? launch_stats<bf16, true>(*d, stream) : launch_stats<bf16, false>(*d, stream);
}

int mmt_distill_grad(const MmtDistill* d, void* stream) {
  if (wrong(*d)) return -2;
  if (d->places == 0) return 0;
  if (d->is_f32) return dual(*d) ? launch_grad<float, true>(*d, stream) : launch_grad<float, false>(*d, stream);
  return dual(*d) ? launch_grad<bf16, true>(*d, stream) : launch_grad<bf16, false>(*d, stream);
}

int mmt_distill_loss(const MmtDistill* d, float* loss, void* stream) {
  if (wrong(*d)) return -2;
  return (int)launch_dependent(distill_loss_kernel, 1, kLossThreads, 0, VR_STREAM(stream), rows_of(*d), call_of(*d), d->rows,
                               d->stats, loss);
}

// n values at a 16-byte boundary.
int mmt_distill_scale(void* grad, int is_f32, long n, const float* factor, void* stream) {
  if (n == 0) return 0;
  const long vecs = (n + 7) / 8, want = (vecs + 255) / 256, most = 8L * mmt_sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  return is_f32 ? (int)launch_dependent(distill_scale_kernel<float>, grid, 256, 0, VR_STREAM(stream),
                                        reinterpret_cast<float*>(grad), n, factor)
                : (int)launch_dependent(distill_scale_kernel<bf16>, grid, 256, 0, VR_STREAM(stream),
                                        reinterpret_cast<bf16*>(grad), n, factor);
}

}  // extern "C"
