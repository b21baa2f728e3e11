// Rows of vocabulary logits: what the kernels for a second model beside the first share (top logits of a teacher,
// distillation from them, verification of drafted tokens).
//
// A row is read in 16-byte vectors that start on 16-byte boundaries, wherever the row itself starts: vector i holds the
// columns i * kVec - lead ... and the first and the last one may be partial.  Odd vocabularies, column slices and padded
// rows then need no copy; only the partial vectors are read element by element.
#pragma once

#include "common.cuh"
#include "runtime.h"

typedef __nv_bfloat16 bf16;

MMT_DEVICE float to_float(float x) { return x; }
MMT_DEVICE float to_float(bf16 x) { return __bfloat162float(x); }
MMT_DEVICE void from_float(float x, float* p) { *p = x; }
MMT_DEVICE void from_float(float x, bf16* p) { *p = __float2bfloat16_rn(x); }

template <typename T>
struct RowVec;
template <>
struct RowVec<bf16> {
  static constexpr int kVec = 8;
  static constexpr uint32_t kNone = 0xff80u;      // -inf
  static MMT_DEVICE uint32_t bits(bf16 x) { return __bfloat16_as_ushort(x); }
  static MMT_DEVICE void unpack(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
  static MMT_DEVICE uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                      pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct RowVec<float> {
  static constexpr int kVec = 4;
  static constexpr uint32_t kNone = 0xff800000u;
  static MMT_DEVICE uint32_t bits(float x) { return __float_as_uint(x); }
  static MMT_DEVICE void unpack(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
  }
  static MMT_DEVICE uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

// One row of V columns.
template <typename T>
struct Row {
  static constexpr int kVec = RowVec<T>::kVec;
  const T* p;
  int V, lead;

  MMT_DEVICE Row(const T* p_, int V_) : p(p_), V(V_), lead(lead_of(p_)) {}
  static MMT_DEVICE int lead_of(const T* q) { return (int)((reinterpret_cast<uintptr_t>(q) & 15) / sizeof(T)); }
  MMT_DEVICE int vectors() const { return (lead + V + kVec - 1) / kVec; }
  MMT_DEVICE int column(int i) const { return i * kVec - lead; }                 // of the first element of vector i
  MMT_DEVICE bool whole(int i) const { return column(i) >= 0 && column(i) + kVec <= V; }
  // Vector i; columns that the row does not have read as -inf.
  MMT_DEVICE uint4 load(int i) const {
    const int c = column(i);
    if (whole(i)) return *reinterpret_cast<const uint4*>(p + c);
    // a first or last vector: not unrolled, which costs the others no registers
    constexpr int kHalf = kVec / 2, kBits = 64 / kHalf;
    unsigned long long half[2] = {0ull, 0ull};
#pragma unroll 1
    for (int j = kVec - 1; j >= 0; --j) {
      const unsigned long long e = c + j >= 0 && c + j < V ? RowVec<T>::bits(p[c + j]) : RowVec<T>::kNone;
      if (j >= kHalf) half[1] = half[1] << kBits | e;
      else half[0] = half[0] << kBits | e;
    }
    return make_uint4((uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32));
  }
  template <typename O>
  static MMT_DEVICE int lead_for(const O* out) { return (int)(reinterpret_cast<uintptr_t>(out) / sizeof(O) % kVec); }
  template <typename O>
  static MMT_DEVICE void store_whole(O* to, const float (&v)[kVec]) {
    if constexpr (sizeof(O) == sizeof(T)) *reinterpret_cast<uint4*>(to) = RowVec<T>::pack(v);
    else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
  // Writes the columns of vector i to the row `out`, of this type or a narrower one, whose start (`out_lead` elements behind
  // a boundary of kVec of them) may lie otherwise.
  template <typename O>
  MMT_DEVICE void store(O* out, int out_lead, int i, const float (&v)[kVec]) const {
    const int c = column(i);
    if (whole(i) && out_lead == lead) {
      store_whole(out + c, v);
      return;
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (c + j >= 0 && c + j < V) from_float(v[j], out + c + j);
  }
};

// ----------------------------------------------------------------------------
// Small arithmetic
// ----------------------------------------------------------------------------
MMT_DEVICE float pow2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
MMT_DEVICE float thread_max(const uint4& u, float m, bf16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) t = __hmax2(t, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
  return fmaxf(m, fmaxf(__low2float(t), __high2float(t)));
}
MMT_DEVICE float thread_max(const uint4& u, float m, float) {
  return fmaxf(fmaxf(m, fmaxf(__uint_as_float(u.x), __uint_as_float(u.y))),
               fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
// Largest of a warp's values, NaN left out.
MMT_DEVICE float warp_top(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Two fp32 values in one 64-bit register: an instruction works on both.
typedef unsigned long long f32x2;
MMT_DEVICE f32x2 both(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
MMT_DEVICE float2 apart(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
MMT_DEVICE f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
MMT_DEVICE f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
MMT_DEVICE f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

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
  // The logit of a key, if the key tells.
  static MMT_DEVICE bool back(uint32_t key, bf16& x) {
    x = __ushort_as_bfloat16((unsigned short)(key & 0x8000u ? key & 0x7fffu : ~key));
    return key != 0x8000u && key != 0xffffu;
  }
  // The largest of a vector's keys, and the upper 16 bits of it.
  static MMT_DEVICE uint32_t top(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) t = __hmax2_nan(t, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    return of(__hmax_nan(__low2bfloat16(t), __high2bfloat16(t)));
  }
  static MMT_DEVICE uint32_t top16(const uint4& u) { return top(u); }
};
template <>
struct Key<float> {
  static constexpr int kBits = 32;
  static MMT_DEVICE uint32_t of(float x) {
    uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;          // one below the largest: there is a key above it
    if (b == 0x80000000u) b = 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static MMT_DEVICE bool back(uint32_t key, float& x) {
    x = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    return key != 0x80000000u && key != 0xfffffffeu;
  }
  static MMT_DEVICE uint32_t top(const uint4& u) {
    return max(max(of(__uint_as_float(u.x)), of(__uint_as_float(u.y))), max(of(__uint_as_float(u.z)), of(__uint_as_float(u.w))));
  }
  static MMT_DEVICE uint32_t top16(const uint4& u) { return top(u) >> 16; }
};

// Element j (of as many as a vector has) of a vector.
template <typename T>
MMT_DEVICE T element(const uint4& v, int j);
template <>
MMT_DEVICE bf16 element<bf16>(const uint4& v, int j) {
  const uint32_t w = j & 4 ? (j & 2 ? v.w : v.z) : (j & 2 ? v.y : v.x);
  return __ushort_as_bfloat16((unsigned short)(j & 1 ? w >> 16 : w));
}
template <>
MMT_DEVICE float element<float>(const uint4& v, int j) {
  return __uint_as_float(j & 2 ? (j & 1 ? v.w : v.z) : (j & 1 ? v.y : v.x));
}

// Sum / maximum over a block of kThreads; `red` holds kThreads / 32 values and may be used again at once.
template <int kThreads, typename F>
MMT_DEVICE F block_total(F v, F* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  F t = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) t += red[w];
  return t;
}
template <int kThreads>
MMT_DEVICE float block_top(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) t = fmaxf(t, red[w]);
  return t;
}

// ----------------------------------------------------------------------------
// Clusters of CTAs that share a row
// ----------------------------------------------------------------------------
MMT_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
MMT_DEVICE uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// All threads of all CTAs of the cluster; shared-memory writes in front of it are seen behind it, in every CTA.
MMT_DEVICE void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Writes to the place in CTA `rank`'s shared memory that `p` has in this CTA's.
MMT_DEVICE void cluster_store(float4* p, uint32_t rank, float4 v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
// Writes to the place in CTA `rank`'s shared memory that `p` has in this CTA's, and counts the 16 bytes into the mbarrier
// there that `bar` is here.
MMT_DEVICE void cluster_send(float4* p, uint64_t* bar, uint32_t rank, float4 v) {
  uint32_t a, b;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(a),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(b)
               : "memory");
}

// Reads the place in CTA `rank`'s shared memory that `p` has in this CTA's.
MMT_DEVICE unsigned long long cluster_load(const unsigned long long* p, uint32_t rank) {
  uint32_t a;
  unsigned long long v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

// mbar_wait (common.cuh) for what other CTAs of the cluster have sent.
MMT_DEVICE bool cluster_wait(uint64_t* bar, uint32_t parity, MmtErrorWord* ew, int where) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t"
        "}\n"
        : "=r"(ok)
        : "r"(addr), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 0x3ff) == 0x3ff) {
      const uint64_t now = mmt_globaltimer();
      if (t0 == 0) t0 = now;
      else if (now - t0 > MMT_WAIT_NS) {
        mmt_report(ew, MMT_ERR_MBAR_TIMEOUT, where, (int)parity);
        return false;
      }
    }
  }
}

// launch_dependent with clusters of `cluster` neighbouring blocks.
template <typename... Params, typename... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), dim3 grid, dim3 block, unsigned cluster, size_t smem,
                           cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Clusters of a kernel that the current device holds at once.
template <typename... Params>
int resident_clusters(void (*kernel)(Params...), unsigned block, unsigned cluster, size_t smem) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = mmt_sm_count() / (int)cluster;
  }
  return n;
}

#define VR_STREAM(s) reinterpret_cast<cudaStream_t>(s)
