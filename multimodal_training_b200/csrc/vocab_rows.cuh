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
  static MMT_DEVICE bf16 none() { return __ushort_as_bfloat16(0xff80); }      // -inf
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
  static MMT_DEVICE float none() { return -INFINITY; }
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
    alignas(16) T e[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      e[j] = RowVec<T>::none();
      if (c + j >= 0 && c + j < V) e[j] = p[c + j];
    }
    return *reinterpret_cast<const uint4*>(e);
  }
  // Writes the columns of vector i to the row `out`, whose start (`out_lead`) may lie otherwise between two boundaries.
  MMT_DEVICE void store(T* out, int out_lead, int i, const float (&v)[kVec]) const {
    const int c = column(i);
    if (whole(i) && out_lead == lead) {
      *reinterpret_cast<uint4*>(out + c) = RowVec<T>::pack(v);
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

#define VR_STREAM(s) reinterpret_cast<cudaStream_t>(s)
