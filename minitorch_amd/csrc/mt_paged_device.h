// Device code that the paged attention kernels share: page resolution, the
// online softmax of a lane group, row chunks and queries in registers, and the
// staging, transposed reads and matrix products of the matrix-core kernels.
#pragma once
#include "mt_device.h"
#include <cmath>
#include <cstdint>

namespace mt {

constexpr int kWave = 64;
constexpr int kGroup = 4;  // lanes per token where a kernel does not say otherwise
constexpr float kLog2e = 1.4426950408889634f;

struct Geometry {
  int heads, dim, page_size, log2_page, pps, num_slabs, columns, layer;
  int64_t kind_stride;  // elements between the K and V planes of one layer
  // p / pps for 0 <= p < 2^31 as (p * pps_magic) >> pps_shift, so that page
  // resolution needs no division: pps_magic = ceil(2^(31+s) / pps) with
  // s = ceil(log2 pps), pps_shift = 31 + s (the error n * e / 2^(31+s),
  // e < 1, stays below 1 / pps for n < 2^31 since pps <= 2^s).
  uint64_t pps_magic;
  int pps_shift;
};

__device__ __forceinline__ int slab_index(int physical, const Geometry& g) {
  return int((uint64_t(uint32_t(physical)) * g.pps_magic) >> g.pps_shift);
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Address of (slot, head, row 0, col 0) in the K plane of `layer`, or nullptr
// for the cases the reference treats as a missing page
// (src/paged_attention_kernel.cu:11-16): logical column out of range, negative
// or out-of-pool physical page, or a null slab.
template <class T>
__device__ __forceinline__ const T* page_base(const uint64_t* slabs, const int* table_row,
                                              int64_t logical, const Geometry& g, int head) {
  if (logical < 0 || logical >= g.columns) return nullptr;
  const int physical = table_row[logical];
  if (physical < 0 || int64_t(physical) >= int64_t(g.num_slabs) * g.pps) return nullptr;
  const int slab = slab_index(physical, g);
  const uint64_t address = slabs[slab];
  if (!address) return nullptr;
  const int slot = physical - slab * g.pps;
  const int64_t i = ((int64_t(g.layer) * 2 * g.pps + slot) * g.heads + head) *
                    int64_t(g.page_size) * g.dim;
  return reinterpret_cast<const T*>(address) + i;
}

// Page base from an already loaded physical page ID (the table read is
// issued separately so that it overlaps other loads).
template <class T>
__device__ __forceinline__ const T* resolve_page(const uint64_t* slabs, int physical,
                                                 const Geometry& g, int head) {
  if (physical < 0 || int64_t(physical) >= int64_t(g.num_slabs) * g.pps) return nullptr;
  const int slab = slab_index(physical, g);
  const uint64_t address = slabs[slab];
  if (!address) return nullptr;
  const int slot = physical - slab * g.pps;
  const int64_t i = ((int64_t(g.layer) * 2 * g.pps + slot) * g.heads + head) *
                    int64_t(g.page_size) * g.dim;
  return reinterpret_cast<const T*>(address) + i;
}

// Page base from a physical page ID and its slab's base address (already
// looked up); nullptr for a null slab.
template <class T>
__device__ __forceinline__ const T* page_in_slab(uint64_t address, int physical, const Geometry& g,
                                                 int head) {
  if (!address) return nullptr;
  const int slot = physical - slab_index(physical, g) * g.pps;
  const int64_t i = ((int64_t(g.layer) * 2 * g.pps + slot) * g.heads + head) *
                    int64_t(g.page_size) * g.dim;
  return reinterpret_cast<const T*>(address) + i;
}

__device__ __forceinline__ bool physical_in_pool(int physical, const Geometry& g) {
  return physical >= 0 && int64_t(physical) < int64_t(g.num_slabs) * g.pps;
}

// Online-softmax state of one token group, in base-2 units (scores are
// pre-multiplied by log2(e)). A missing page contributes a NaN score, which
// fmaxf drops from the running max and which then poisons the denominator,
// matching the reference's NaN propagation (src/paged_attention_kernel.cu:53,66-69,84).
template <int N, int G = kGroup>
struct Softmax {
  float m, l, acc[N];
  __device__ __forceinline__ void init() {
    m = -INFINITY; l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
  }
  __device__ __forceinline__ void add(float s, const float* v) {
    const float mn = fmaxf(m, s);
    const float alpha = (m == -INFINITY) ? 0.f : fast_exp2(m - mn);
    const float p = fast_exp2(s - mn);
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(p, v[i], acc[i] * alpha);
    m = mn;
  }
  // Add U tokens with one rescale: the running max moves once per call.
  template <int U, class VF>
  __device__ __forceinline__ void add_many(const float* s, const bool* valid, VF&& v_of) {
    float mx = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (valid[u]) mx = fmaxf(mx, s[u]);
    const float alpha = (m == -INFINITY) ? 0.f : fast_exp2(m - mx);
    l *= alpha;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (valid[u]) {
        const float p = fast_exp2(s[u] - mx);
        l += p;
        float v[N];
        v_of(u, v);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(p, v[i], acc[i]);
      }
    }
    m = mx;
  }
  __device__ __forceinline__ void merge(float mo, float lo, const float* ao) {
    const float mn = fmaxf(m, mo);
    const float sa = (m == -INFINITY) ? 0.f : fast_exp2(m - mn);
    const float sb = (mo == -INFINITY) ? 0.f : fast_exp2(mo - mn);
    l = l * sa + lo * sb;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = acc[i] * sa + ao[i] * sb;
    m = mn;
  }
  // Merge with the state held `rot` lanes further along the same 16-lane row
  // (DPP row rotate; no LDS traffic).
  template <int CTRL>
  __device__ __forceinline__ void merge_dpp() {
    float ao[N];
    const float mo = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), CTRL, 0xF, 0xF, false));
    const float lo = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(l), CTRL, 0xF, 0xF, false));
#pragma unroll
    for (int i = 0; i < N; ++i)
      ao[i] = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(acc[i]), CTRL, 0xF, 0xF, false));
    merge(mo, lo, ao);
  }
  // Merge the token groups of each 16-lane row: afterwards lanes with
  // lane % 16 < G hold their row's state for chunk lane % G.
  __device__ __forceinline__ void row_merge() {
    static_assert(G == 4 || G == 8, "row_merge expects 4 or 8 lanes per token");
    if constexpr (G == 4) merge_dpp<0x124>();  // row_ror:4
    merge_dpp<0x128>();                        // row_ror:8
  }
  // Merge the states of the token groups of a wave (lanes with equal
  // lane % G): afterwards lanes 0..G-1 hold the wave's state for their chunk.
  __device__ __forceinline__ void wave_merge() {
#pragma unroll
    for (int off = G; off < kWave; off <<= 1) {
      float ao[N];
      const float mo = __shfl_xor(m, off);
      const float lo = __shfl_xor(l, off);
#pragma unroll
      for (int i = 0; i < N; ++i) ao[i] = __shfl_xor(acc[i], off);
      merge(mo, lo, ao);
    }
  }
};

__device__ __forceinline__ float finalize(float acc, float l) {
  return l > 0.f ? acc / l : (isnan(l) ? NAN : 0.f);
}

// Sum of a value over the G lanes of a token group with DPP: quad permutes
// for 4 lanes, then the half-row mirror (lane i <-> 7 - i) for 8 lanes.
template <int G = kGroup>
__device__ __forceinline__ float group_sum(float x) {
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, true));
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, true));
  if constexpr (G == 8)
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xF, 0xF, true));
  return x;
}

// How a decode reads rows: element by element, masked to the head dim; in
// 16-byte loads when the head dim is the kernel's (64 or 128); in 16-byte
// loads masked to a smaller head dim of whole 16-byte chunks (80 of 128, 32 of
// 64), whose other lanes hold zeros.
enum Rows : int { kRowsElements = 0, kRowsFull = 1, kRowsPadded = 2 };

// Per-lane chunk of one token row: DL values at `p` (K or V plane), converted
// to fp32. VEC (Rows) uses 16-byte loads; otherwise element loads masked to `dim`.
// The G lanes of a row take its 16-byte chunks in turn (lane g chunks g, g + G,
// ..), so that each load instruction covers consecutive bytes also where a lane
// owns several chunks; with a lane's chunks next to each other fp32 and head
// dim 128 streamed at 2.1-2.8 TB/s, fp32's 8 x 900 tokens x 25 heads of 128 in
// 64 us. col_of(i): the column of a lane's value i less its first.
template <int DT, int DL, int VEC, int G>
struct Chunk {
  static __device__ __forceinline__ constexpr int col_of(int i) {
    return VEC ? i / per16<DT>() * (G * per16<DT>()) + i % per16<DT>() : i;
  }
  static __device__ __forceinline__ int first_col(int g) { return VEC ? g * per16<DT>() : g * DL; }
  using T = typename Elem<DT>::T;
  static constexpr int NV = VEC ? DL * elem_bytes<DT>() / 16 : 1;
  u32x4 raw[VEC ? NV : 1];
  float val[VEC ? 1 : DL];
  // NTL: non-temporal loads (data read once, not kept in the caches).
  template <bool NTL = false>
  __device__ __forceinline__ void load(const T* p, int col0, int dim) {
    if constexpr (VEC) {
      const auto* v = global_view(reinterpret_cast<const u32x4*>(p));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (VEC == kRowsPadded && col0 + i * G * per16<DT>() >= dim) raw[i] = u32x4{0u, 0u, 0u, 0u};
        else if constexpr (NTL) raw[i] = __builtin_nontemporal_load(v + i * G);
        else raw[i] = v[i * G];
      }
    } else {
      const auto* g = global_view(p);
#pragma unroll
      for (int i = 0; i < DL; ++i) val[i] = (col0 + i < dim) ? to_f32<DT>(g[i]) : 0.f;
    }
  }
  // Same chunk from an LDS copy of the row (p points at column col0).
  __device__ __forceinline__ void load_lds(const T* p, int col0, int dim) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i] = reinterpret_cast<const u32x4*>(p)[i * G];
    } else {
#pragma unroll
      for (int i = 0; i < DL; ++i) val[i] = (col0 + i < dim) ? to_f32<DT>(p[i]) : 0.f;
    }
  }
  __device__ __forceinline__ void nan_fill() {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i] = u32x4{~0u, ~0u, ~0u, ~0u};
    } else {
#pragma unroll
      for (int i = 0; i < DL; ++i) val[i] = NAN;
    }
  }
  __device__ __forceinline__ void to_float(float* o) const {
    if constexpr (VEC) {
      constexpr int E = per16<DT>();
#pragma unroll
      for (int i = 0; i < NV; ++i) unpack16<DT>(raw[i], o + i * E);
    } else {
#pragma unroll
      for (int i = 0; i < DL; ++i) o[i] = val[i];
    }
  }
};

// One query vector split over the 4 lanes of a token group. For fp16/bf16
// with 16-byte access the query stays packed in its input type and q.k uses
// the fp32-accumulating dot2 instructions (v_dot2c_f32_f16 / _bf16), so no
// K conversion is needed and the query takes DL/2 registers; the 1/sqrt(D)
// and log2(e) factors are applied to the summed score. fp32 and the masked
// path keep a pre-scaled fp32 query.
template <int DT, int D, int VEC, int G = kGroup>
struct Query {
  using T = typename Elem<DT>::T;
  static constexpr int DL = D / G;
  static constexpr bool PACKED = VEC && DT != kF32;
  uint32_t qp[PACKED ? DL / 2 : 1];
  float qf[PACKED ? 1 : DL];
  float post_scale;
  __device__ __forceinline__ void load(const T* q, int col0, int dim, float scale) {
    Chunk<DT, DL, VEC, G> c;
    c.load(q + col0, col0, dim);
    if constexpr (PACKED) {
#pragma unroll
      for (int w = 0; w < DL / 2; ++w) qp[w] = c.raw[w / 4][w % 4];
      post_scale = scale;
    } else {
      c.to_float(qf);
#pragma unroll
      for (int i = 0; i < DL; ++i) qf[i] *= scale;
      post_scale = 1.f;
    }
  }
  // This lane's part of q.k (before the group sum and post_scale).
  __device__ __forceinline__ float partial(const Chunk<DT, DL, VEC, G>& k) const {
    float s = 0.f;
    if constexpr (PACKED) {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int w = 0; w < DL / 2; ++w) {
        const uint32_t kw = k.raw[w / 4][w % 4];
        if constexpr (DT == kF16)
          s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, qp[w]), __builtin_bit_cast(h2, kw), s, false);
        else
          s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, qp[w]), __builtin_bit_cast(b2, kw), s, false);
      }
    } else {
      float kf[DL];
      k.to_float(kf);
#pragma unroll
      for (int i = 0; i < DL; ++i) s = fmaf(qf[i], kf[i], s);
    }
    return s;
  }
  __device__ __forceinline__ float score(const Chunk<DT, DL, VEC, G>& k) const {
    return group_sum<G>(partial(k)) * post_scale;
  }
};

// x of lanes l and l ^ 32 (in either order): the permlane swap of two copies
// of x leaves x[l % 32] in one and x[l % 32 + 32] in the other.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Two probabilities as the high and low packed MFMA operands: hi = p rounded
// to the input type (fp16 toward zero, one packed conversion; bf16 to nearest
// even), lo = the remainder, rounded the same way.
template <int DT>
struct SplitP;
template <>
struct SplitP<kF16> {
  static __device__ __forceinline__ void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(p0, p1);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0 - float(h[0]), p1 - float(h[1])));
  }
};
template <>
struct SplitP<kBF16> {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const bf2 h = {static_cast<__bf16>(p0), static_cast<__bf16>(p1)};
    hi = __builtin_bit_cast(uint32_t, h);
    asm("" : "+v"(hi));  // keeps the halves' unpacking from becoming two more conversions
    const float r0 = p0 - __uint_as_float(hi << 16), r1 = p1 - __uint_as_float(hi & 0xffff0000u);
    const bf2 r = {static_cast<__bf16>(r0), static_cast<__bf16>(r1)};
    lo = __builtin_bit_cast(uint32_t, r);
  }
};

typedef float floatx16 __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ floatx16 mfma32(const u32x4& x, const u32x4& y, const floatx16& c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Mfma<kF16>::v8, x),
                                                  __builtin_bit_cast(Mfma<kF16>::v8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Mfma<kBF16>::v8, x),
                                                   __builtin_bit_cast(Mfma<kBF16>::v8, y), c, 0, 0, 0);
}

// Four keys of one dim: lane t of each 16 lanes passes row t / 4, columns
// 4 (t % 4) .. + 3 of a 4 x 16 block of 16-bit elements and receives column t.
__device__ __forceinline__ uint2 read_transposed(const void* p) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  const s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
  return __builtin_bit_cast(uint2, r);
}

// acc / l by the output rule (0 for l = 0, NaN for a NaN l) with inv =
// inverse(l): one multiplication for 16-bit results, corrected to fp32's
// rounding for fp32 ones.
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : (isnan(l) ? NAN : 0.f); }
template <int DT>
__device__ __forceinline__ float divided(float acc, float l, float inv) {
  const float x = acc * inv;
  if constexpr (DT == kF32) return fabsf(x) < INFINITY ? fmaf(fmaf(-x, l, acc), inv, x) : x;
  else return x;
}

// What a staged row reads where there is nothing to read: NaN keys (a missing
// page: its scores are NaN) and zeros, each a 16-byte load.
static __device__ __align__(16) const uint32_t g_fill[8] = {~0u, ~0u, ~0u, ~0u, 0u, 0u, 0u, 0u};

// Copies 16 bytes per lane from global memory to LDS without passing through
// registers: lane l's bytes land at lds + 16 l. The compiler does not see the
// write, nor count it in its own waits: wait_staged() before the barrier that
// publishes a round.
__device__ __forceinline__ void stage16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "m0", "memory");
}
__device__ __forceinline__ void stage16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" ::"s"(base), "v"(offset), "s"(lds)
               : "m0", "memory");
}
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t x = reinterpret_cast<uintptr_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(x)), hi = __builtin_amdgcn_readfirstlane(uint32_t(x >> 32));
  return reinterpret_cast<const char*>(uint64_t(hi) << 32 | lo);
}
// Waits until at most N of this wave's memory operations are outstanding.
template <int N>
__device__ __forceinline__ void wait_staged() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

inline Geometry make_geometry(int h, int d, int page_size, int pps, int num_slabs, int columns, int layer) {
  Geometry g{};
  g.heads = h; g.dim = d; g.page_size = page_size;
  g.log2_page = page_size == 8 ? 3 : page_size == 16 ? 4 : 5;
  g.pps = pps; g.num_slabs = num_slabs; g.columns = columns; g.layer = layer;
  int sh = 0;
  while ((int64_t(1) << sh) < pps) ++sh;
  g.pps_shift = 31 + sh;
  g.pps_magic = ((uint64_t(1) << (31 + sh)) + uint64_t(pps) - 1) / uint64_t(pps);
  g.kind_stride = int64_t(pps) * h * page_size * d;
  return g;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Compute units of the current device (cached per device).
inline int device_compute_units() {
  static int cached[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  if (!cached[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cached[dev] = n;
  }
  return cached[dev];
}

}  // namespace mt
