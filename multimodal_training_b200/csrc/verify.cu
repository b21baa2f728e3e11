// Verification of drafted tokens against the target model's logits from given random numbers.
//
// A sequence has drafts x_0 .. x_{len-1}; row i of the target holds the logits behind which x_i was drafted, row len those
// behind the last of them.  With p_i = softmax(target_i / tau) and q_i = softmax(draft_i / tau) (without draft logits: all
// mass on x_i), x_i is accepted while u_i q_i(x_i) < p_i(x_i), up to the first place a where that fails.  The next token
// is drawn from max(p_a - q_a, 0), from p_a where that has no mass, or from p_len when all are accepted: the smallest id
// whose cumulative weight exceeds r times the total.  tau = 0: x_i is accepted while it is the largest logit's id (equal
// logits: the lowest id, NaN above everything), and the next token is that id of row a.
//
// A drawn token depends on a sum over the whole vocabulary that may end next to a border, so probabilities and sums are
// fp64: an error e of the cumulative weights gives another token with probability 2 V e.
#include "vocab_rows.cuh"

namespace {

constexpr int kVerifyThreads = 512;

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
  double* stats;                      // [batch, 2 drafts + 1, 2]: largest logit and sum of exp((x - largest) / tau);
                                      // without sampling the id of the largest logit
  double inv_temperature;
  int batch, drafts, V, is_f32, uniforms_f64, sampled;
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
MMT_DEVICE double weight(float x, double top, double inv_temperature) {
  return exp(((double)x - top) * inv_temperature);
}

// ----------------------------------------------------------------------------
// Rows: largest logit and normaliser, or the id of the largest logit.  One CTA per row: the drafts + 1 of the target, then
// those of the draft model.
// ----------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_rows_kernel(Verify v) {
  grid_dependency_sync();
  __shared__ float red[kVerifyThreads / 32];
  __shared__ double dred[kVerifyThreads / 32];
  const int b = blockIdx.y, r = blockIdx.x, len = draft_len(v, b);
  const bool of_target = r <= v.drafts;
  if (of_target ? r > len : r - v.drafts - 1 >= len) return;
  const Row<T> row = of_target ? target_row<T>(v, b, r) : draft_row<T>(v, b, r - v.drafts - 1);
  const int nv = row.vectors();
  double* out = v.stats + ((long)b * (2 * v.drafts + 1) + r) * 2;
  float m = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < nv; i += kVerifyThreads) {
    float x[Row<T>::kVec];
    RowVec<T>::unpack(row.load(i), x);
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j) {
      m = fmaxf(m, x[j]);
      nan |= !(x[j] == x[j]);
    }
  }
  m = block_top<kVerifyThreads>(m, red);
  if (!v.sampled) {
    nan = __syncthreads_or(nan);
    __shared__ int first;
    if (threadIdx.x == 0) first = v.V;
    __syncthreads();
    int mine = v.V;
    for (int i = threadIdx.x; i < nv && mine == v.V; i += kVerifyThreads) {
      float x[Row<T>::kVec];
      RowVec<T>::unpack(row.load(i), x);
      const int c = row.column(i);
#pragma unroll
      for (int j = Row<T>::kVec - 1; j >= 0; --j)
        if (c + j >= 0 && c + j < v.V && (nan ? !(x[j] == x[j]) : x[j] == m)) mine = c + j;
    }
    if (mine < v.V) atomicMin(&first, mine);
    __syncthreads();
    if (threadIdx.x == 0) out[0] = (double)first;
    return;
  }
  double s = 0.0;
  for (int i = threadIdx.x; i < nv; i += kVerifyThreads) {
    float x[Row<T>::kVec];
    RowVec<T>::unpack(row.load(i), x);
    const int c = row.column(i);
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j)
      if (c + j >= 0 && c + j < v.V) s += weight(x[j], (double)m, v.inv_temperature);
  }
  s = block_total<kVerifyThreads>(s, dred);
  if (threadIdx.x == 0) {
    out[0] = (double)m;
    out[1] = s;
  }
}

// Accepted drafts of a sequence; the first `drafts` entries of accept_prob and the tokens but the drawn one.
template <typename T>
MMT_DEVICE int accept(const Verify& v, int b, int len, int* first) {
  if (threadIdx.x == 0) *first = len;
  __syncthreads();
  const double* st = v.stats + (long)b * (2 * v.drafts + 1) * 2;
  for (int i = threadIdx.x; i < v.drafts; i += kVerifyThreads) {
    float prob = 0.f;
    if (i < len) {
      const long x = v.draft_ids[(long)b * v.drafts + i];
      bool ok;
      if (!v.sampled) {
        ok = (double)x == st[2 * i];
        prob = ok ? 1.f : 0.f;
      } else {
        double p = 0.0, q = v.draft ? 0.0 : 1.0;
        if (x >= 0 && x < v.V) {
          p = weight(to_float(target_row<T>(v, b, i).p[x]), st[2 * i], v.inv_temperature) / st[2 * i + 1];
          const double* sd = st + 2 * (v.drafts + 1 + i);
          if (v.draft) q = weight(to_float(draft_row<T>(v, b, i).p[x]), sd[0], v.inv_temperature) / sd[1];
        }
        ok = uniform(v, b, i) * q < p;
        prob = p > 0.0 ? (p >= q ? 1.f : (float)(p / q)) : p == 0.0 ? 0.f : NAN;
      }
      if (!ok) atomicMin(first, i);
    }
    v.accept_prob[(long)b * v.drafts + i] = prob;
  }
  __syncthreads();
  const int a = *first;
  for (int i = threadIdx.x; i <= v.drafts; i += kVerifyThreads)
    if (i != a) v.tokens[(long)b * (v.drafts + 1) + i] = i < a ? v.draft_ids[(long)b * v.drafts + i] : -1;
  if (threadIdx.x == 0) v.accepted[b] = a;
  return a;
}

// ----------------------------------------------------------------------------
// Sequences: acceptance, then the next token.  One CTA per sequence; every thread draws from one run of vectors.
// ----------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_draw_kernel(Verify v) {
  grid_dependency_sync();
  __shared__ int first;
  __shared__ double part[kVerifyThreads];
  __shared__ int chosen, last;
  const int b = blockIdx.x, len = draft_len(v, b), tid = threadIdx.x;
  const int a = accept<T>(v, b, len, &first);
  const double* st = v.stats + (long)b * (2 * v.drafts + 1) * 2;
  long* token = v.tokens + (long)b * (v.drafts + 1) + a;
  if (!v.sampled) {
    if (tid == 0) *token = (long)st[2 * a];
    return;
  }
  const Row<T> p = target_row<T>(v, b, a);
  const bool rejected = a < len;
  const long x = rejected ? v.draft_ids[(long)b * v.drafts + a] : -1;
  const double* sp = st + 2 * a;
  const double* sq = st + 2 * (v.drafts + 1 + a);
  const T* q = rejected && v.draft ? draft_row<T>(v, b, a).p : nullptr;
  const double top_p = sp[0], sum_p = sp[1], top_q = q ? sq[0] : 0.0, sum_q = q ? sq[1] : 1.0;
  const int nv = p.vectors(), per = (nv + kVerifyThreads - 1) / kVerifyThreads;
  bool rest = rejected;                      // weights are max(p - q, 0); false: p
  auto weigh = [&](int c, float xp) {
    const double w = weight(xp, top_p, v.inv_temperature) / sum_p;
    if (!rest) return w;
    if (q == nullptr) return c == x ? 0.0 : w;
    const double d = w - weight(to_float(q[c]), top_q, v.inv_temperature) / sum_q;
    return d > 0.0 ? d : 0.0;
  };
  double total;
  for (;;) {
    double s = 0.0;
    for (int i = tid * per; i < min((tid + 1) * per, nv); ++i) {
      float e[Row<T>::kVec];
      RowVec<T>::unpack(p.load(i), e);
      const int c = p.column(i);
#pragma unroll
      for (int j = 0; j < Row<T>::kVec; ++j)
        if (c + j >= 0 && c + j < v.V) s += weigh(c + j, e[j]);
    }
    __syncthreads();
    part[tid] = s;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kVerifyThreads; ++i) part[i] += part[i - 1];
      chosen = v.V;
      last = -1;
    }
    __syncthreads();
    total = part[kVerifyThreads - 1];
    if (total > 0.0 || !rest) break;
    rest = false;
  }
  const double goal = uniform(v, b, v.drafts) * total;
  const double before = tid ? part[tid - 1] : 0.0;
  double s = 0.0;
  int mine = v.V, end = -1;
  if (part[tid] > before)
    for (int i = tid * per; i < min((tid + 1) * per, nv); ++i) {
      float e[Row<T>::kVec];
      RowVec<T>::unpack(p.load(i), e);
      const int c = p.column(i);
#pragma unroll
      for (int j = 0; j < Row<T>::kVec; ++j) {
        if (c + j < 0 || c + j >= v.V) continue;
        const double w = weigh(c + j, e[j]);
        s += w;
        if (w > 0.0) end = c + j;
        if (w > 0.0 && before + s > goal && mine == v.V) mine = c + j;
      }
    }
  atomicMin(&chosen, mine);
  atomicMax(&last, end);
  __syncthreads();
  // by rounding the goal may lie behind the last sum; no id has any weight if the target's row is not a distribution
  if (tid == 0) *token = chosen < v.V ? chosen : last;
}

template <typename T>
int launch_verify(const Verify& v, void* stream) {
  const int rows = v.sampled && v.draft ? 2 * v.drafts + 1 : v.drafts + 1;
  const int e = (int)launch_dependent(verify_rows_kernel<T>, dim3(rows, v.batch), kVerifyThreads, 0, VR_STREAM(stream), v);
  if (e) return e;
  return (int)launch_dependent(verify_draw_kernel<T>, v.batch, kVerifyThreads, 0, VR_STREAM(stream), v);
}

}  // namespace

extern "C" {

int mmt_verify_bytes() { return (int)sizeof(Verify); }

int mmt_verify_drafts(const void* words, void* stream) {
  const Verify& v = *reinterpret_cast<const Verify*>(words);
  if (v.batch < 0 || v.batch > 65535 || v.drafts < 0 || v.drafts > 65535 || v.V < 1) return -2;
  if (v.batch == 0) return 0;
  return v.is_f32 ? launch_verify<float>(v, stream) : launch_verify<bf16>(v, stream);
}

}  // extern "C"
