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
  // Writes the columns of vector i to the row `out`, of this type or a narrower one, whose start (`out_lead` elements behind
  // a boundary of kVec of them) may lie otherwise.
  template <typename O>
  static MMT_DEVICE int lead_for(const O* out) { return (int)(reinterpret_cast<uintptr_t>(out) / sizeof(O) % kVec); }
  template <typename O>
  static MMT_DEVICE void store_whole(O* to, const float (&v)[kVec]) {
    if constexpr (sizeof(O) == sizeof(T)) *reinterpret_cast<uint4*>(to) = RowVec<T>::pack(v);
    else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
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
