// The global norm of many gradient tensors, and their clipping by it (no counterpart in the reference, whose optimizer step is
// autolabel/trainer.py:45-48 without one):
//     norm = sqrt(sum over tensors and elements of g^2) / loss_scale,   g <- g min(1, max_norm / (norm + 1e-6))
// Two launches per list of up to CLIP_LIST tensors, whatever their sizes and types: k_grad_sumsq leaves one partial sum per block,
// k_grad_scale adds the partial sums up again in every one of its blocks (8 KB from L2, always in the same order: every block arrives at the
// same bits, with no atomic and no third launch) and scales.  Squares and sums are fp64: an fp32 gradient's square overflows fp32 from 1.8e19 on,
// and the fp64 multiply-add is free beside the loads that bound both kernels.
#include "common.h"
#include <algorithm>
#include <new>
#include <vector>

#define CLIP_LIST 120        // tensors per launch: their table travels as the kernel's argument (under 4 KB), so a captured graph holds it too
#define CLIP_CHUNK 8192      // elements a block takes at a time
#define CLIP_BLOCKS 1024     // four blocks per CU at most: enough loads in flight, and few partial sums
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
enum { FT_F16 = 0, FT_BF16 = 1, FT_F32 = 2 };
struct ClipList {
  const void* g[CLIP_LIST]; void* o[CLIP_LIST]; int64_t n[CLIP_LIST];
  int32_t first[CLIP_LIST + 1];    // first chunk of a tensor
  uint8_t type[CLIP_LIST];
  int32_t count;
};
struct ClipRule { float max_norm; const float* loss_scale; float* norm; int32_t* found_inf; const double* part; int32_t parts; };

// The chunk's tensor (the last one whose first chunk is not behind it; tensors without elements have no chunk).
__device__ inline int clip_find(const ClipList& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1; }
  return lo;
}
template <int T> __device__ inline void load8(const void* p, int64_t at, float (&v)[8]) {
  if constexpr (T == FT_F32) __builtin_memcpy(v, (const float*)p + at, 32);
  else {
    u16x8 w;
    __builtin_memcpy(&w, (const uint16_t*)p + at, 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = T == FT_F16 ? (float)__builtin_bit_cast(h16, (uint16_t)w[j]) : __uint_as_float((uint32_t)w[j] << 16);
  }
}
template <int T> __device__ inline float load1(const void* p, int64_t at) {
  if constexpr (T == FT_F32) return ((const float*)p)[at];
  else if constexpr (T == FT_F16) return (float)((const h16*)p)[at];
  else return __uint_as_float((uint32_t)((const uint16_t*)p)[at] << 16);
}
template <int T> __device__ inline void store1(void* p, int64_t at, float v) {
  if constexpr (T == FT_F32) ((float*)p)[at] = v;
  else if constexpr (T == FT_F16) ((h16*)p)[at] = (h16)v;
  else ((__bf16*)p)[at] = (__bf16)v;
}
__device__ inline double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// the sum over the 256 threads of a block, in every one of them
__device__ inline double block_sum_d(double v, double* lds4) {
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) lds4[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds4[0] + lds4[1]) + (lds4[2] + lds4[3]);
}

template <int T> __device__ inline double sumsq_chunk(const void* g, int64_t lo, int64_t hi) {
  double s = 0.0, t = 0.0;
  int64_t i = lo + threadIdx.x * 8;
#pragma unroll 4
  for (; i + 8 <= hi; i += 2048) {
    float v[8];
    load8<T>(g, i, v);
#pragma unroll
    for (int j = 0; j < 8; j += 2) { s += (double)v[j] * (double)v[j]; t += (double)v[j + 1] * (double)v[j + 1]; }
  }
  if (i < hi) for (; i < hi; ++i) { const double v = load1<T>(g, i); s += v * v; }
  return s + t;
}
__global__ __launch_bounds__(256) void k_grad_sumsq(ClipList l, double* part) {
  __shared__ double lds4[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < l.first[l.count]; c += gridDim.x) {
    const int k = clip_find(l, c);
    const int64_t lo = (int64_t)(c - l.first[k]) * CLIP_CHUNK, hi = min(lo + CLIP_CHUNK, l.n[k]);
    s += l.type[k] == FT_F32 ? sumsq_chunk<FT_F32>(l.g[k], lo, hi) : l.type[k] == FT_F16 ? sumsq_chunk<FT_F16>(l.g[k], lo, hi) : sumsq_chunk<FT_BF16>(l.g[k], lo, hi);
  }
  s = block_sum_d(s, lds4);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// NT: what goes to another buffer passes the caches by, so that the gradients just squared are still there (36 -> 33 us for the 14.8 M
// parameters of a field with 512-wide heads).
template <int T, bool NT> __device__ inline void scale_chunk(const void* g, void* o, int64_t lo, int64_t hi, float f, float p2) {
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));
  int64_t i = lo + threadIdx.x * 8;
#pragma unroll 4
  for (; i + 8 <= hi; i += 2048) {
    float v[8];
    load8<T>(g, i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * f * p2;
    if constexpr (T == FT_F32) {
      const f32x4u a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
      f32x4u* p = (f32x4u*)((float*)o + i);
      if (NT) { __builtin_nontemporal_store(a, p); __builtin_nontemporal_store(b, p + 1); }
      else { p[0] = a; p[1] = b; }
    } else {
      u16x8u w;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = T == FT_F16 ? __builtin_bit_cast(uint16_t, (h16)v[j]) : __builtin_bit_cast(uint16_t, (__bf16)v[j]);
      u16x8u* p = (u16x8u*)((uint16_t*)o + i);
      if (NT) __builtin_nontemporal_store(w, p);
      else *p = w;
    }
  }
  if (i < hi) for (; i < hi; ++i) store1<T>(o, i, load1<T>(g, i) * f * p2);
}
template <int T> __device__ inline void scale_chunk(const void* g, void* o, int64_t lo, int64_t hi, float f, float p2) {
  if (g == o) scale_chunk<T, false>(g, o, lo, hi, f, p2);
  else scale_chunk<T, true>(g, o, lo, hi, f, p2);
}
__global__ __launch_bounds__(256) void k_grad_scale(ClipList l, ClipRule r, int apply, int in_place) {
  __shared__ double lds4[4];
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < r.parts; i += 256) s += r.part[i];
  double norm = sqrt(block_sum_d(s, lds4));
  if (r.loss_scale) norm /= (double)*r.loss_scale;
  const bool finite = fabs(norm) <= 3.4028234663852886e38;
  // a norm that is not finite scales nothing: the caller skips the step (found_inf), and the gradients show where it came from
  const double ratio = finite ? fmin(1.0, (double)r.max_norm / (norm + 1e-6)) : 1.0;
  // (a factor near or under fp32's least normal keeps its bits as f 2^-100: v f does not overflow, f <= 1, and the power of two is exact)
  const bool low = ratio < 0x1p-100;
  const float f = (float)(low ? ratio * 0x1p100 : ratio), p2 = low ? 0x1p-100f : 1.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (r.norm) *r.norm = (float)norm;
    if (r.found_inf && !finite) *r.found_inf = 1;
  }
  if (!apply || (in_place && f == 1.f && !low)) return;
  // backwards: what was squared last is the likeliest to be in the caches still
  const int total = l.first[l.count], grid = gridDim.x;
  for (int c = (total - 1) / grid * grid + (int)blockIdx.x; c >= 0; c -= grid) {
    if (c >= total) continue;
    const int k = clip_find(l, c);
    const int64_t lo = (int64_t)(c - l.first[k]) * CLIP_CHUNK, hi = min(lo + CLIP_CHUNK, l.n[k]);
    if (l.type[k] == FT_F32) scale_chunk<FT_F32>(l.g[k], l.o[k], lo, hi, f, p2);
    else if (l.type[k] == FT_F16) scale_chunk<FT_F16>(l.g[k], l.o[k], lo, hi, f, p2);
    else scale_chunk<FT_BF16>(l.g[k], l.o[k], lo, hi, f, p2);
  }
}

struct Span { uintptr_t lo, hi; };
// true when two of the spans share a byte
static bool spans_meet(std::vector<Span>& s) {
  std::sort(s.begin(), s.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  for (size_t i = 1; i < s.size(); ++i) if (s[i].lo < s[i - 1].hi) return true;
  return false;
}

extern "C" int64_t aln_grad_clip_ws_bytes(int32_t n) { return n > 0 ? ((int64_t)n + CLIP_LIST - 1) / CLIP_LIST * CLIP_BLOCKS * 8 : 0; }
extern "C" int aln_grad_clip(int32_t n, const void* const* grads, void* const* out, const int64_t* numel, const int32_t* types, float max_norm, int32_t apply,
                             const float* loss_scale, float* norm, int32_t* found_inf, void* ws, int64_t ws_bytes, void* stream) {
  ALN_REQUIRE(n >= 1 && grads && numel && types, "grad_clip: an empty list of tensors");
  ALN_REQUIRE(max_norm >= 0.f, "grad_clip: max_norm = %g", (double)max_norm);
  ALN_REQUIRE(ws && ((uintptr_t)ws & 7) == 0 && ws_bytes >= aln_grad_clip_ws_bytes(n), "grad_clip: the workspace needs %lld bytes, aligned to 8", (long long)aln_grad_clip_ws_bytes(n));
  try {
    std::vector<Span> from, to;
    from.reserve(n); to.reserve(n + 3);
    for (int k = 0; k < n; ++k) {
      ALN_REQUIRE(types[k] >= FT_F16 && types[k] <= FT_F32, "grad_clip: tensor %d has the unknown type %d", k, types[k]);
      ALN_REQUIRE(numel[k] >= 0 && numel[k] < (int64_t)1 << 40, "grad_clip: tensor %d has %lld elements", k, (long long)numel[k]);
      if (numel[k] == 0) continue;
      const int es = types[k] == FT_F32 ? 4 : 2;
      ALN_REQUIRE(grads[k] && ((uintptr_t)grads[k] & (es - 1)) == 0, "grad_clip: tensor %d is NULL or not aligned to its type", k);
      from.push_back({(uintptr_t)grads[k], (uintptr_t)grads[k] + numel[k] * es});
      if (!apply || !out || out[k] == grads[k]) continue;
      ALN_REQUIRE(out[k] && ((uintptr_t)out[k] & (es - 1)) == 0, "grad_clip: output %d is NULL or not aligned to its type", k);
      to.push_back({(uintptr_t)out[k], (uintptr_t)out[k] + numel[k] * es});
    }
    if (apply) {    // what is scaled must not be read again by another block of the same launch
      to.insert(to.end(), from.begin(), from.end());
      for (const void* w : {(const void*)loss_scale, (const void*)norm, (const void*)found_inf}) if (w) to.push_back({(uintptr_t)w, (uintptr_t)w + 4});
      ALN_REQUIRE(!spans_meet(to), "grad_clip: two of the tensors share memory");
    }
  } catch (const std::bad_alloc&) {
    aln_set_error("grad_clip: out of host memory");
    return -1;
  }
  hipStream_t st = (hipStream_t)stream;
  const int lists = (n + CLIP_LIST - 1) / CLIP_LIST;
  ClipRule r{max_norm, loss_scale, norm, found_inf, (const double*)ws, 0};
  for (int pass = 0; pass < 2; ++pass) {
    int parts = 0;
    for (int a = 0; a < lists; ++a) {
      ClipList l{};
      bool in_place = true;
      for (int k = a * CLIP_LIST; k < n && k < (a + 1) * CLIP_LIST; ++k) {
        if (numel[k] == 0) continue;
        const int i = l.count++;
        l.g[i] = grads[k]; l.o[i] = out ? out[k] : const_cast<void*>(grads[k]); l.n[i] = numel[k]; l.type[i] = (uint8_t)types[k];
        in_place &= l.o[i] == l.g[i];
        const int64_t end = l.first[i] + (numel[k] + CLIP_CHUNK - 1) / CLIP_CHUNK;
        ALN_REQUIRE(end < (int64_t)1 << 31, "grad_clip: too many elements");
        l.first[i + 1] = (int32_t)end;
      }
      const int blocks = aln_grid_for(l.first[l.count], 1, CLIP_BLOCKS);
      if (pass == 0) { hipLaunchKernelGGL(k_grad_sumsq, dim3(blocks), dim3(256), 0, st, l, (double*)ws + parts); parts += blocks; }
      else if (a == 0 || apply) {
        hipLaunchKernelGGL(k_grad_scale, dim3(apply ? blocks : 1), dim3(256), 0, st, l, r, apply, (int)in_place);
        r.norm = nullptr; r.found_inf = nullptr;
      }
      ALN_CHECK_LAUNCH("grad_clip");
    }
    if (pass == 0) r.parts = parts;
  }
  return 0;
}
