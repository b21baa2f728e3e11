// Verification of drafted tokens against the target model's logits from given random numbers.
//
// A sequence has drafts x_0 .. x_{len-1}; row i of the target holds the logits behind which x_i was drafted, row len those
// behind the last of them.  With p_i = softmax(target_i / tau) and q_i = softmax(draft_i / tau) (without draft logits: all
// mass on x_i), x_i is accepted while u_i q_i(x_i) < p_i(x_i), up to the first place a where that fails.  The next token
// is drawn from max(p_a - q_a, 0), from p_a where that has no mass, or from p_len when all are accepted: the smallest id
// whose cumulative weight exceeds r times the total.  tau = 0: x_i is accepted while it is the largest logit's id (equal
// logits: the lowest id, NaN above everything), and the next token is that id of row a.
//
// A drawn token depends on a sum over the whole vocabulary that may end next to a border: an error e of the cumulative
// weights gives another token with probability 2 V e.  So the row that is drawn from is weighed in fp64.  The normalisers of
// all rows, one pass over memory, are fp32 sums of a bounded error (sum_error), so a draft whose acceptance that could change
// has its two rows summed again in fp64.
#include "vocab_rows.cuh"

namespace {

constexpr int kRowThreads = 256;                  // of a CTA that reads a part of a row
constexpr int kRowAhead = 4;                      // vectors that a thread loads before it works on them
constexpr int kDrawThreads = 256;                 // two CTAs an SM, with up to 128 registers a thread
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kDrawCluster = 16;                  // most CTAs that weigh a row
constexpr double kLog2e = 1.44269504088896340736;

struct Verify {
  const void* target;                 // [batch, drafts + 1, V]
  const void* draft;                  // [batch, drafts, V] or null
  long target_seq, target_row, draft_seq, draft_row;      // strides in elements
  const long* draft_ids;              // [batch, drafts]
  const void* uniforms;               // [batch, drafts + 1], fp32 or fp64; null without sampling
  const long* lens;                   // [batch] or null
  long* accepted;                     // [batch]
  long* tokens;                       // [batch, drafts + 1]
  float* accept_prob;                 // [batch, drafts]
  unsigned long long* parts;          // [batch, rows, splits]: (largest logit, sum of 2^((x - largest) c)) of each part of
                                      // a row; without sampling the key of its largest logit
  double inv_temperature;
  int batch, drafts, V, is_f32, uniforms_f64, sampled;
  int rows, splits;                   // rows of a sequence (the target's, then the draft model's), parts of a row
};

MMT_DEVICE int draft_len(const Verify& v, int b) {
  if (v.lens == nullptr) return v.drafts;
  const long n = v.lens[b];
  return (int)(n < 0 ? 0 : n > v.drafts ? v.drafts : n);
}
MMT_DEVICE double uniform(const Verify& v, int b, int i) {
  const long at = (long)b * (v.drafts + 1) + i;
  return v.uniforms_f64 ? reinterpret_cast<const double*>(v.uniforms)[at]
                        : (double)reinterpret_cast<const float*>(v.uniforms)[at];
}
template <typename T>
MMT_DEVICE Row<T> target_row(const Verify& v, int b, int i) {
  return Row<T>(reinterpret_cast<const T*>(v.target) + b * v.target_seq + i * v.target_row, v.V);
}
template <typename T>
MMT_DEVICE Row<T> draft_row(const Verify& v, int b, int i) {
  return Row<T>(reinterpret_cast<const T*>(v.draft) + b * v.draft_seq + i * v.draft_row, v.V);
}
// fp32 exponents are (x - m) c, as in the sums of csrc/distill.cu.
MMT_DEVICE float scale_of(const Verify& v) { return (float)(kLog2e * v.inv_temperature); }

// Bound on the relative error of a row's fp32 sum, in which a thread adds kRowAhead vectors a step.  In units of 2^-24: a step
// may scale what there is by another power (four for ex2.approx, one for the product) and adds to it (one); besides those a
// term's power (four) and its exponent, whose three roundings count in proportion to it, 20.8 on the average of a
// distribution over 2^30 ids; 16 additions of a step and 15 of the threads, warps and their scales.
MMT_DEVICE double sum_error(const Verify& v) {
  const int vec = v.is_f32 ? 4 : 8, per = (v.V / vec + v.splits) / v.splits + 1;
  return (6.0 * ((per - 1) / (kRowAhead * kRowThreads) + 1) + 100.0) * 0x1p-24;
}

// ----------------------------------------------------------------------------
// Rows: (largest logit, sum), or the key of the largest logit, of each part of a row.  One pass over memory: 139 MB (the rows
// of 48 sequences with up to five drafts, 152064 columns in bf16) in 30 us, 4.6 TB/s.
// ----------------------------------------------------------------------------
template <typename T>
MMT_DEVICE unsigned long long key_of(T x, int c) {
  return (unsigned long long)Key<T>::of(x) << 32 | (0xffffffffu - (uint32_t)c);
}

template <typename T, bool kSampled>
__global__ void __launch_bounds__(kRowThreads) verify_rows_kernel(Verify v) {
  grid_dependency_sync();
  constexpr int kVec = Row<T>::kVec, kWarps = kRowThreads / 32;
  __shared__ float2 warp_part[kWarps];
  __shared__ unsigned long long warp_key[kWarps];
  const int b = blockIdx.z, r = blockIdx.y, len = draft_len(v, b);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool of_target = r <= v.drafts;
  if (of_target ? r > len : r - v.drafts - 1 >= len) return;
  const Row<T> row = of_target ? target_row<T>(v, b, r) : draft_row<T>(v, b, r - v.drafts - 1);
  // vectors [first, stop) of the row, whole ones [lo, hi); `edge`: a column outside the whole ones for each of a few threads
  const int nv = row.vectors(), per = (nv + v.splits - 1) / v.splits;
  const int first = blockIdx.x * per, stop = min(first + per, nv);
  const int lo = first + (first == 0 && row.lead != 0), hi = max(lo, min(stop, (row.lead + v.V) / kVec));
  int edge = -1;
  if (first < stop) {
    const int head = max(row.column(first), 0), head_end = min(row.column(min(lo, stop)), v.V);
    const int tail = max(row.column(hi), 0), tail_end = min(row.column(stop), v.V);
    if (head + tid < head_end) edge = head + tid;
    else if (tid >= kVec && tail + tid - kVec < tail_end) edge = tail + tid - kVec;
  }
  unsigned long long* out = v.parts + ((long)b * v.rows + r) * v.splits + blockIdx.x;

  if constexpr (!kSampled) {
    // a thread's largest vector, the first of several; its element is looked up in the end
    uint32_t top = 0;
    int at = -1;
    for (int i0 = lo + tid; i0 < hi; i0 += kRowAhead * kRowThreads) {
      uint4 u[kRowAhead];
#pragma unroll
      for (int k = 0; k < kRowAhead; ++k)
        if (i0 + k * kRowThreads < hi) u[k] = *reinterpret_cast<const uint4*>(row.p + row.column(i0 + k * kRowThreads));
#pragma unroll
      for (int k = 0; k < kRowAhead; ++k) {
        const int i = i0 + k * kRowThreads;
        const uint32_t t = i < hi ? Key<T>::top(u[k]) : 0;
        if (t > top) {
          top = t;
          at = i;
        }
      }
    }
    unsigned long long key = edge >= 0 ? key_of(row.p[edge], edge) : 0;
    if (at >= 0) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) key = max(key, key_of(row.p[row.column(at) + j], row.column(at) + j));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if (lane == 0) warp_key[warp] = key;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kWarps; ++w) key = max(key, warp_key[w]);
      *out = key;
    }
  } else {
    const float c = scale_of(v);
    const f32x2 c2 = both(c, c);
    const float x0 = edge >= 0 ? to_float(row.p[edge]) : -INFINITY;
    float m = warp_top(x0);
    // what is not a number makes the sum so, and a warp that has nothing but -inf adds zeros (2^-inf), not 2^(-inf + inf)
    f32x2 s = both(edge >= 0 ? pow2((x0 - (m == -INFINITY ? 0.f : m)) * c) : 0.f, 0.f);
    for (int i0 = lo + warp * 32; i0 < hi; i0 += kRowAhead * kRowThreads) {
      uint4 u[kRowAhead];
      const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
      for (int k = 0; k < kRowAhead; ++k) {
        const int i = i0 + k * kRowThreads + lane;
        u[k] = make_uint4(none, none, none, none);
        if (i < hi) u[k] = *reinterpret_cast<const uint4*>(row.p + row.column(i));
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kRowAhead; ++k) top = thread_max(u[k], top, T());
      top = warp_top(top);
      if (top > m) {
        const float by = m == -INFINITY ? 0.f : pow2((m - top) * c);
        s = mul2(s, both(by, by));
        m = top;
      }
      const float less = m == -INFINITY ? 0.f : m;
      const f32x2 less2 = both(-less, -less);
      f32x2 few = both(0.f, 0.f);                  // of these vectors: 16 terms, which keeps the chain of roundings short
#pragma unroll
      for (int k = 0; k < kRowAhead; ++k) {
        float x[kVec];
        RowVec<T>::unpack(u[k], x);
#pragma unroll
        for (int j = 0; j < kVec; j += 2) {
          const float2 e = apart(mul2(add2(both(x[j], x[j + 1]), less2), c2));
          few = add2(few, both(pow2(e.x), pow2(e.y)));
        }
      }
      s = add2(s, few);
    }
    const float sum = warp_sum(apart(s).x + apart(s).y);
    if (lane == 0) warp_part[warp] = make_float2(m, sum);
    __syncthreads();
    if (warp == 0) {
      const float2 a = warp_part[lane % kWarps];
      const float top = warp_top(a.x);
      float part = a.x == -INFINITY ? a.y : a.y * pow2((a.x - top) * c);
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == 0) *reinterpret_cast<float2*>(out) = make_float2(top, part);
    }
  }
}

// ----------------------------------------------------------------------------
// Sequences.  The first CTA of a sequence's cluster writes its answers.  A rejected draft costs four fp64 powers a column: two
// for the rows' sums, two for max(p - q, 0); an accepted one nothing, and the row behind the last one power.  Those powers
// bound it: 64 us for the 48 sequences above, half of the issue slots and a third of the fp64 pipe.  A sequence by itself is a
// chain of barriers: 22 us with its rows.  256 threads of 128 registers: 87 us with the rows, 512 of 64: 95, three CTAs of 256
// an SM: 97.  Half as many CTAs again as fill the SMs once: 107 instead of 95, both with 512 threads.
// ----------------------------------------------------------------------------
constexpr int kChunk = 32;            // drafts that are looked at together
enum Verdict { kStands, kHangs, kFalls };
struct DrawShared {
  double table[16];                   // 2^(i / 16)
  double warp_total[kDrawWarps];
  float4 cta_part[2][kDrawCluster];   // two doubles each
  int verdict[kChunk];                // of a chunk of drafts: stands, hangs on the sums' errors, falls
  float2 logits[kChunk], largest[kChunk];     // of the draft, and of its rows (the target's, the draft model's)
};

// 2^(x scale / 16 - whole / 16) in fp64, for a whole number `whole` near the largest x scale of the row: x scale - whole = n + f
// with a whole n and |f| <= 1/2; 2^(n / 16) from a table of 16 (one word of each bank: no conflicts) and the exponent, 2^(f / 16)
// by its series, whose rest is 2e-13 of it (Tang, Table-driven implementation of the exponential function, 1989).  Nine fp64
// instructions and no branches: what bounds the drawn rows is how many instructions a power takes.  The row is a distribution:
// its largest logit is finite and none is not a number.  Logits 900 powers of two below the largest, -inf too, count as that
// far below, which is nothing (kNothing).
struct Powers16 {
  static constexpr double kMagic = 6755399441055744.0;    // 1.5 * 2^52: a number near it is rounded to a whole one
  double scale, shift, largest;                   // shift = kMagic - whole
  float least;
  MMT_DEVICE Powers16(double scale_, double largest_)
      : scale(scale_), shift(kMagic - rint(largest_ * scale_)), largest(largest_),
        least((float)(largest_ - 16.0 * 900.0 / scale_)) {}
  // Whether the largest logit is too far from zero for `least`, whose rounding to fp32 moves it by 2^-24 of that distance: up to
  // here that is 64 of the 900 powers of two, and what is left is between 2^-964, where the exponent still fits, and 2^-836,
  // which is nothing.  Rows further out take the long way.  (Beside kMagic a whole number has room up to 2^51.)
  MMT_DEVICE bool far() const { return fabs(largest) * scale > 0x1p34; }
  MMT_DEVICE double any(float x, const double* table) const {
    return far() ? exp2(((double)x - largest) * (scale / 16.0)) : of(x, table);
  }
  MMT_DEVICE double of(float x, const double* table) const {
    constexpr double L = 0.69314718055994530942 / 16.0, L2 = L * L;
    const double d = (double)fmaxf(x, least), shifted = fma(d, scale, shift), f = fma(d, scale, shift - shifted);
    const int n = __double2loint(shifted);
    double p = fma(L2 * L2 * L / 120.0, f, L2 * L2 / 24.0);
    p = fma(p, f, L2 * L / 6.0);
    p = fma(p, f, L2 / 2.0);
    p = fma(p, f, L);
    const double t = table[n & 15], e = fma(t, p * f, t);
    return __hiloint2double(__double2hiint(e) + ((n >> 4) << 20), __double2loint(e));
  }
};

// Weights of the columns of a row that a token is drawn from.
constexpr double kNothing = 0x1p-800;             // a weight or a sum that is none
constexpr double kNoRest = 0x1p-46;               // a sum of max(p - q, 0) that may be the rounding of p and q, 2^-53 a step
enum Draw { kPlain, kWithout, kRest };            // p; p without one id; max(p - q, 0)
template <typename T>
struct Weigher {
  Row<T> p;
  const T* q;
  const double* table;
  Powers16 of_p, of_q;
  double by_p, by_q;
  long x;
  Draw kind;
  MMT_DEVICE double rest(T xp, T xq) const {
    const double d = of_p.of(to_float(xp), table) * by_p - of_q.of(to_float(xq), table) * by_q;
    return d > 0.0 ? d : 0.0;
  }
  MMT_DEVICE double of(T xp, int c) const {
    const double e = of_p.any(to_float(xp), table);
    if (kind != kRest) return kind == kWithout && c == x ? 0.0 : e;
    const double d = e * by_p - of_q.any(to_float(q[c]), table) * by_q;
    return d > 0.0 ? d : 0.0;
  }
  // Sum over vector i, whose logits are `u` if it is a whole one.
  MMT_DEVICE double sum(int i, const uint4& u) const {
    const int c = p.column(i);
    double s = 0.0;
    if (p.whole(i) && !of_p.far() && !of_q.far()) {
      if (kind == kRest && Row<T>::lead_of(q) == p.lead) {
        const uint4 uq = *reinterpret_cast<const uint4*>(q + c);
#pragma unroll
        for (int j = 0; j < Row<T>::kVec; ++j) s += rest(element<T>(u, j), element<T>(uq, j));
      } else if (kind != kRest) {
#pragma unroll
        for (int j = 0; j < Row<T>::kVec; ++j) {
          const double e = of_p.of(to_float(element<T>(u, j)), table);
          s += kind == kWithout && c + j == x ? 0.0 : e;
        }
      } else {
#pragma unroll 1
        for (int j = 0; j < Row<T>::kVec; ++j) s += rest(element<T>(u, j), q[c + j]);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < Row<T>::kVec; ++j)
        if (c + j >= 0 && c + j < p.V) s += of(p.p[c + j], c + j);
    }
    return s;
  }
  // Sum over the vectors from `i` on in steps of `step`, below `stop`.
  MMT_DEVICE double sum_run(int i, int stop, int step) const {
    double s = 0.0;
    uint4 next = make_uint4(0u, 0u, 0u, 0u);
    if (i < stop && p.whole(i)) next = *reinterpret_cast<const uint4*>(p.p + p.column(i));
    for (; i < stop; i += step) {
      const uint4 u = next;
      if (i + step < stop && p.whole(i + step)) next = *reinterpret_cast<const uint4*>(p.p + p.column(i + step));
      s += sum(i, u);
    }
    return s;
  }
};

MMT_DEVICE double warp_total_of(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 2) verify_draw_kernel(Verify v) {
  grid_dependency_sync();
  __shared__ DrawShared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int b = blockIdx.x / C, n = v.drafts, len = draft_len(v, b);
  const long at = (long)b * (n + 1);
  if (tid < 16) s.table[tid] = exp2((double)tid / 16.0);
  __syncthreads();
  cluster_barrier();                               // every CTA has started: its shared memory may be written
  int turn = 0;
  const double scale = 16.0 * kLog2e * v.inv_temperature;      // of Powers16
  // what p / q may be off by, twice over: 2^-13 up to 550,000 columns (270,000 in fp32) in one part
  const double margin = 1.0 + fmax(4.0 * sum_error(v), 0x1p-13);

  // largest logit and normaliser of a row, from its parts; by a warp
  const float c = scale_of(v);
  auto row_sum = [&](int r) {
    const float2* part = reinterpret_cast<const float2*>(v.parts + ((long)b * v.rows + r) * v.splits);
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 x = lane < v.splits ? part[lane] : none, y = lane + 32 < v.splits ? part[lane + 32] : none;
    const float m = warp_top(fmaxf(x.x, y.x));
    auto of = [&](float2 p) {
      return p.x == -INFINITY ? (double)p.y : (double)p.y * exp2(((double)p.x - (double)m) * (double)c);
    };
    return make_double2((double)m, warp_total_of(of(x) + of(y)));
  };
  // largest logit's id of a row without sampling; by a warp
  auto row_choice = [&](int r) {
    const unsigned long long* part = v.parts + ((long)b * v.rows + r) * v.splits;
    unsigned long long key = max(lane < v.splits ? part[lane] : 0ull, lane + 32 < v.splits ? part[lane + 32] : 0ull);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    return (long)(0xffffffffu - (uint32_t)key);
  };
  // a value of each CTA, summed in their order
  auto cluster_total = [&](double2 mine) {
    if (tid < C) {
      float4 w;
      *reinterpret_cast<double2*>(&w) = mine;
      cluster_store(&s.cta_part[turn][rank], tid, w);
    }
    cluster_barrier();
    double2 total = make_double2(0.0, 0.0);
    for (int k = 0; k < C; ++k) {
      const double2 a = *reinterpret_cast<const double2*>(&s.cta_part[turn][k]);
      total.x += a.x;
      total.y += a.y;
    }
    turn ^= 1;
    return total;
  };
  auto block_sum = [&](double x) {
    x = warp_total_of(x);
    __syncthreads();
    if (lane == 0) s.warp_total[warp] = x;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kDrawWarps; ++w) t += s.warp_total[w];
    return t;
  };
  // this CTA's run of a row's vectors
  auto run_of = [&](const Row<T>& row) {
    const int nv = row.vectors(), per = (nv + C - 1) / C;
    return make_int2(min(rank * per, nv), min((rank + 1) * per, nv));
  };
  // normalisers of a row of the target and of the draft model, in fp64 (relative to the largest logits as Powers16 has them)
  auto exact_sums = [&](int i, bool with_q, double m_p, double m_q) {
    Weigher<T> w = {target_row<T>(v, b, i), nullptr, s.table, Powers16(scale, m_p), Powers16(scale, m_p), 1.0, 1.0, -1, kPlain};
    int2 run = run_of(w.p);
    const double sum_p = block_sum(w.sum_run(run.x + tid, run.y, kDrawThreads));
    double sum_q = 0.0;
    if (with_q) {
      w.p = draft_row<T>(v, b, i);
      w.of_p = Powers16(scale, m_q);
      run = run_of(w.p);
      sum_q = block_sum(w.sum_run(run.x + tid, run.y, kDrawThreads));
    }
    return cluster_total(make_double2(sum_p, sum_q));
  };

  // ---- acceptance: every CTA decides for itself
  int a = len;
  for (int c0 = 0; c0 < len; c0 += kChunk) {
    const int in_chunk = min(kChunk, len - c0);
    for (int j = warp; j < in_chunk; j += kDrawWarps) {
      const int i = c0 + j;
      const long x = v.draft_ids[(long)b * n + i];
      float prob;
      int verdict;
      if (!v.sampled) {
        verdict = x == row_choice(i) ? kStands : kFalls;
        prob = verdict == kStands ? 1.f : 0.f;
      } else {
        const bool known = x >= 0 && x < v.V;
        const double2 sp = row_sum(i), sq = v.draft ? row_sum(n + 1 + i) : make_double2(0.0, 1.0);
        const float xp = known ? to_float(target_row<T>(v, b, i).p[x]) : 0.f;
        const float xq = known && v.draft ? to_float(draft_row<T>(v, b, i).p[x]) : 0.f;
        auto share = [&](float x, double2 sum) { return exp2(((double)x - sum.x) * (scale / 16.0)) / sum.y; };
        const double p = known ? share(xp, sp) : 0.0, q = !v.draft ? 1.0 : known ? share(xq, sq) : 0.0;
        const double uq = uniform(v, b, i) * q;
        prob = p > 0.0 ? (p >= q ? 1.f : (float)(p / q)) : p == 0.0 ? 0.f : NAN;
        verdict = uq * margin < p ? kStands : uq < p * margin && p > 0.0 ? kHangs : kFalls;
        if (lane == 0) {
          s.logits[j] = make_float2(xp, xq);
          s.largest[j] = make_float2((float)sp.x, (float)sq.x);
        }
      }
      if (lane == 0) {
        s.verdict[j] = verdict;
        if (rank == 0) v.accept_prob[(long)b * n + i] = prob;
      }
    }
    __syncthreads();
    for (int j = 0; j < in_chunk && a == len; ++j) {
      bool falls = s.verdict[j] == kFalls;
      if (s.verdict[j] == kHangs) {
        const float2 x = s.logits[j], m = s.largest[j];
        const double2 sums = exact_sums(c0 + j, v.draft != nullptr, m.x, m.y);
        const double q = v.draft ? Powers16(scale, m.y).any(x.y, s.table) / sums.y : 1.0;
        falls = !(uniform(v, b, c0 + j) * q < Powers16(scale, m.x).any(x.x, s.table) / sums.x);
      }
      if (falls) a = c0 + j;
    }
    __syncthreads();
  }
  if (rank == 0) {
    for (int i = len + tid; i < n; i += kDrawThreads) v.accept_prob[(long)b * n + i] = 0.f;
    for (int i = tid; i <= n; i += kDrawThreads)
      if (i != a) v.tokens[at + i] = i < a ? v.draft_ids[(long)b * n + i] : -1;
    if (tid == 0) v.accepted[b] = a;
  }
  long* token = v.tokens + at + a;
  if (!v.sampled) {
    const long choice = row_choice(a);
    if (rank == 0 && tid == 0) *token = choice;
    return;
  }

  // ---- the next token
  // a row of the target that is no distribution draws nothing, one of the draft model leaves the target's
  const double2 of_row = row_sum(a), of_draft = a < len && v.draft ? row_sum(n + 1 + a) : make_double2(0.0, 1.0);
  const double m_p = of_row.x, m_q = of_draft.x;
  auto distribution = [](double2 r) { return fabs(r.x) < INFINITY && r.y > 0.0 && r.y < INFINITY; };
  const bool sound = distribution(of_row);
  Weigher<T> w = {target_row<T>(v, b, a), nullptr, s.table, Powers16(scale, m_p), Powers16(scale, m_p), 1.0, 1.0, -1, kPlain};
  if (a < len && sound && distribution(of_draft)) {
    w.kind = kWithout;
    w.x = v.draft_ids[(long)b * n + a];
    if (v.draft) {
      const double2 sums = exact_sums(a, true, m_p, m_q);
      w.kind = kRest;
      w.q = draft_row<T>(v, b, a).p;
      w.of_q = Powers16(scale, m_q);
      w.by_p = 1.0 / sums.x;
      w.by_q = 1.0 / sums.y;
    }
  }
  // a warp weighs a run of neighbouring vectors
  const int2 run = run_of(w.p);
  const int share = (run.y - run.x + kDrawWarps - 1) / kDrawWarps;
  auto warp_run = [&](int k) { return make_int2(min(run.x + k * share, run.y), min(run.x + (k + 1) * share, run.y)); };
  double rest = 0.0;                               // weight up to the token, from this CTA's first vector on
  int owner = -1;
  while (sound) {
    const int2 mine = warp_run(warp);
    const double part = block_sum(w.sum_run(mine.x + lane, mine.y, 32));
    const double total = cluster_total(make_double2(part, 0.0)).x;
    if (!(total > (w.kind == kRest ? kNoRest : kNothing))) {
      if (w.kind == kPlain) break;
      w.kind = kPlain;                              // no mass but the draft's: from the target itself
      continue;
    }
    // the first CTA whose weights pass the goal; by rounding the goal may lie behind all: the last one with any weight
    const double goal = uniform(v, b, n) * total;
    double up_to = 0.0;
    for (int k = 0; k < C && !(owner >= 0 && up_to > goal); ++k) {
      const double x = reinterpret_cast<const double2*>(&s.cta_part[turn ^ 1][k])->x;
      if (!(x > kNothing)) continue;
      owner = k;
      rest = goal - up_to;
      up_to += x;
    }
    break;
  }
  if (owner < 0 && rank == 0 && tid == 0) *token = -1;      // the target's row is no distribution
  if (owner != rank) return;
  // the same among the runs of this CTA's warps, and among as many parts of the one that it is
  auto pick = [&](int2 whole, int part) {
    int k = -1;
    double up_to = 0.0, from = 0.0;
    for (int q = 0; q < kDrawWarps && !(k >= 0 && up_to > rest); ++q) {
      const double x = s.warp_total[q];
      if (!(x > kNothing)) continue;
      k = q;
      from = up_to;
      up_to += x;
    }
    rest -= from;
    k = max(k, 0);
    return make_int2(min(whole.x + k * part, whole.y), min(whole.x + (k + 1) * part, whole.y));
  };
  const int2 coarse = pick(run, share);
  const int finer = (coarse.y - coarse.x + kDrawWarps - 1) / kDrawWarps;
  const int from = min(coarse.x + warp * finer, coarse.y), to = min(from + finer, coarse.y);
  (void)block_sum(w.sum_run(from + lane, to, 32));
  const int2 fine = pick(coarse, finer);
  if (warp != 0) return;
  for (int i0 = fine.x; i0 < fine.y; i0 += 32) {
    double x = w.sum_run(i0 + lane, min(fine.y, i0 + lane + 1), 1), up_to = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, up_to, o);
      if (lane >= o) up_to += y;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, up_to > rest && x > kNothing);
    if (past) {
      // this vector: a lane weighs a column
      const int who = __ffs(past) - 1;
      const double before = __shfl_sync(0xffffffffu, up_to - x, who);
      const int col = w.p.column(i0 + who) + lane;
      const double y = lane < Row<T>::kVec && col >= 0 && col < v.V ? w.of(w.p.p[col], col) : 0.0;
      double sum = y;
#pragma unroll
      for (int o = 1; o < Row<T>::kVec; o <<= 1) {
        const double z = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += z;
      }
      const uint32_t weighty = __ballot_sync(0xffffffffu, y > kNothing);
      const uint32_t chosen = __ballot_sync(0xffffffffu, y > kNothing && before + sum > rest);
      // by rounding the goal may lie behind the vector: its last column with any weight
      if (lane == (chosen ? __ffs(chosen) - 1 : 31 - __clz(weighty | 1u))) *token = max(col, 0);
      return;
    }
    rest -= __shfl_sync(0xffffffffu, up_to, 31);
  }
  // by rounding the goal lies behind this part: its last column with any weight
  if (lane == 0) {
    int col = min(w.p.column(fine.y), v.V) - 1;
    const int least = max(w.p.column(fine.x), 0);
    while (col > least && !(w.of(w.p.p[col], col) > kNothing)) --col;
    *token = col;
  }
}

// Parts of a row: enough CTAs for eight an SM, as long as each thread has kRowAhead vectors.
int splits_of(long rows, int V, int is_f32) {
  const long most = V / (is_f32 ? 4 : 8) / (kRowAhead * kRowThreads);
  const long want = (8L * mmt_sm_count() + rows - 1) / (rows > 0 ? rows : 1);
  const long n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

template <typename T>
int launch_verify(const Verify& v, void* stream) {
  const dim3 grid(v.splits, v.rows, v.batch);
  const int e = (int)(v.sampled ? launch_dependent(verify_rows_kernel<T, true>, grid, kRowThreads, 0, VR_STREAM(stream), v)
                                : launch_dependent(verify_rows_kernel<T, false>, grid, kRowThreads, 0, VR_STREAM(stream), v));
  if (e) return e;
  auto kernel = verify_draw_kernel<T>;
  static bool allowed = false;                     // clusters of more than eight
  if (!allowed) {
    const cudaError_t c = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (c != cudaSuccess) return (int)c;
    allowed = true;
  }
  // two CTAs an SM
  const int want = 2 * mmt_sm_count() / v.batch;
  const unsigned C = !v.sampled || want < 1 ? 1 : want < kDrawCluster ? want : kDrawCluster;
  return (int)launch_cluster(kernel, v.batch * C, kDrawThreads, C, 0, VR_STREAM(stream), v);
}

}  // namespace

extern "C" {

int mmt_verify_bytes() { return (int)sizeof(Verify); }
// Parts that `rows` rows of V columns are read in.
int mmt_verify_splits(long rows, int V, int is_f32) { return splits_of(rows, V, is_f32); }

int mmt_verify_drafts(const void* words, void* stream) {
  const Verify& v = *reinterpret_cast<const Verify*>(words);
  if (v.batch < 0 || v.batch > 65535 || v.drafts < 0 || v.rows > 65535 || v.rows < v.drafts + 1 || v.V < 1 || v.splits < 1)
    return -2;
  if (v.batch == 0) return 0;
  return v.is_f32 ? launch_verify<float>(v, stream) : launch_verify<bf16>(v, stream);
}

}  // extern "C"
