// Attention of a batch behind a shared prefix, and the K/V append through a slot
// map, for gfx950 (CDNA4, wave64). Pages, slabs and missing pages as in
// paged_attention_kernel.hip.
#include "mt_paged_device.h"
#include "../../include/mt_shared.h"
#include <algorithm>
#include <climits>

using namespace mt;

namespace {

// ---------------------------------------------------------------------------
// K/V rows to their pages through a slot map. VEC moves 16 bytes per thread.
struct SlotArgs {
  const void* k;
  const void* v;
  const uint64_t* slabs;
  const int64_t* slots;
  int64_t units;  // per-thread units of K (and V)
  int64_t stride;
  Geometry g;
};

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void append_slots_kernel(SlotArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int E = VEC ? per16<DT>() : 1;
  const Geometry& g = a.g;
  const int per_head = g.dim / E, per_row = g.heads * per_head;
  const int64_t slots = int64_t(g.num_slabs) * g.pps * g.page_size;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < a.units; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row;
    const int unit = int(i - row * per_row);
    const int head = unit / per_head, col = (unit - head * per_head) * E;
    const int64_t slot = a.slots[row];
    if (slot < 0 || slot >= slots) continue;
    const T* page = resolve_page<T>(a.slabs, int(slot >> g.log2_page), g, head);
    if (!page) continue;
    T* kp = const_cast<T*>(page) + (int(slot) & (g.page_size - 1)) * g.dim + col;
    T* vp = kp + g.kind_stride;
    const int64_t src = row * a.stride + int64_t(head) * g.dim + col;
    if constexpr (VEC) {
      *global_view(reinterpret_cast<u32x4*>(kp)) = *global_view(reinterpret_cast<const u32x4*>(static_cast<const T*>(a.k) + src));
      *global_view(reinterpret_cast<u32x4*>(vp)) = *global_view(reinterpret_cast<const u32x4*>(static_cast<const T*>(a.v) + src));
    } else {
      *kp = static_cast<const T*>(a.k)[src];
      *vp = static_cast<const T*>(a.v)[src];
    }
  }
}

// ---------------------------------------------------------------------------
// Attention over a shared prefix and a request's own tokens.
struct SharedArgs {
  void* out;
  const void* q;
  const void* k;  // decode: the new tokens' rows (strides of q); null: every key is in the pages
  const void* v;
  const uint64_t* slabs;
  const int* prefix_table;
  const int* table;
  const int* lengths;    // own tokens before the new ones
  const int* cu_tokens;  // null: one new token per request
  int b, rows, max_tokens, prefix;
  float qscale;  // log2(e) / sqrt(d)
  int64_t q_r, o_r;  // elements between rows of q (k, v) and out
  Geometry g;        // columns: of the block table
  int prefix_columns;
};

// The rows of request r: first row, new tokens and own tokens before them
// (sane values whatever the arrays hold).
struct Request {
  int row0, tokens, length;
};
__device__ __forceinline__ Request request_of(const SharedArgs& a, int r) {
  Request q{r, 1, a.lengths[r]};
  if (a.cu_tokens) {
    const int c0 = a.cu_tokens[r], c1 = a.cu_tokens[r + 1];
    q.row0 = min(max(c0, 0), a.rows);
    q.tokens = min(min(max(c1, q.row0), a.rows) - q.row0, a.max_tokens);
  }
  return q;
}

// One wave's walk over keys [k0, k1) of a table row for one query: a lane scores
// every 64th key, then holds columns lane and lane + 64 of the output. The last
// key may come from rows of its own (fresh_k, fresh_v). Any head dim and
// alignment: elements are read one by one.
template <int DT>
struct Walk {
  using T = typename Elem<DT>::T;
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};  // l: this lane's keys

  __device__ __forceinline__ void keys(const T* q, const uint64_t* slabs, const int* table_row, int columns, int64_t k0,
                                       int64_t k1, const T* fresh_k, const T* fresh_v, const Geometry& g, int head,
                                       float qscale) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll 1
    for (int64_t c0 = k0; c0 < k1; c0 += kWave) {
      const int64_t key = c0 + lane;
      const T *kp = nullptr, *vp = nullptr;
      float s = key < k1 ? NAN : -INFINITY;  // a missing page's score is NaN
      if (key < k1) {
        const int64_t column = key >> g.log2_page;
        const T* page = column < columns ? resolve_page<T>(slabs, table_row[column], g, head) : nullptr;
        if (page) {
          const bool fresh = fresh_k && key == k1 - 1;
          kp = fresh ? fresh_k : page + int(key & (g.page_size - 1)) * g.dim;
          vp = fresh ? fresh_v : page + g.kind_stride + int(key & (g.page_size - 1)) * g.dim;
          s = 0.f;
#pragma unroll 1
          for (int c = 0; c < g.dim; ++c) s = fmaf(to_f32<DT>(q[c]), to_f32<DT>(global_view(kp)[c]), s);
          s *= qscale;
        }
      }
      float top = s;
#pragma unroll
      for (int w = kWave / 2; w > 0; w /= 2) top = fmaxf(top, __shfl_xor(top, w));
      top = fmaxf(m, top);
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - top);
      const float p = fast_exp2(s - (top == -INFINITY ? 0.f : top));
      m = top;
      l = fmaf(l, alpha, p);
      acc[0] *= alpha;
      acc[1] *= alpha;
      const uint64_t v_at = reinterpret_cast<uintptr_t>(vp);
      const int n = int(k1 - c0 < kWave ? k1 - c0 : kWave);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
        const T* vj = reinterpret_cast<const T*>(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v_at >> 32), j))) << 32 |
                                                 uint32_t(__builtin_amdgcn_readlane(int(v_at), j)));
        if (!vj) continue;
        if (lane < g.dim) acc[0] = fmaf(pj, to_f32<DT>(global_view(vj)[lane]), acc[0]);
        if (lane + kWave < g.dim) acc[1] = fmaf(pj, to_f32<DT>(global_view(vj)[lane + kWave]), acc[1]);
      }
    }
  }
  __device__ __forceinline__ float denominator() const {
    float x = l;
#pragma unroll
    for (int w = kWave / 2; w > 0; w /= 2) x += __shfl_xor(x, w);
    return x;
  }
};

// One wave per (request, new token, head): right for every shape. The prefix is
// walked once per query here, so this is the path of rows that are not whole,
// aligned 16-byte chunks only.
template <int DT>
__global__ __launch_bounds__(256) void shared_walk_kernel(SharedArgs a) {
  using T = typename Elem<DT>::T;
  const Geometry& g = a.g;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t items = int64_t(a.b) * a.max_tokens * g.heads;
  for (int64_t item = blockIdx.x * 4 + (threadIdx.x >> 6); item < items; item += int64_t(gridDim.x) * 4) {
    const int64_t ri = item / g.heads;
    const int head = int(item - ri * g.heads);
    const int r = int(ri / a.max_tokens), i = int(ri - int64_t(r) * a.max_tokens);
    const Request rq = request_of(a, r);
    if (i >= rq.tokens) continue;
    const int64_t row = rq.row0 + i;
    const T* q = static_cast<const T*>(a.q) + row * a.q_r + int64_t(head) * g.dim;
    T* out = static_cast<T*>(a.out) + row * a.o_r + int64_t(head) * g.dim;
    const int* table_row = a.table + int64_t(r) * g.columns;
    Walk<DT> w;
    if (rq.length >= 0) {
      const int64_t keys = int64_t(rq.length) + i + 1;
      const T *fk = nullptr, *fv = nullptr;
      if (a.k) {
        fk = static_cast<const T*>(a.k) + row * a.q_r + int64_t(head) * g.dim;
        fv = static_cast<const T*>(a.v) + row * a.q_r + int64_t(head) * g.dim;
        const int64_t column = (keys - 1) >> g.log2_page;
        const T* page = column < g.columns ? resolve_page<T>(a.slabs, table_row[column], g, head) : nullptr;
        if (page) {
          T* kp = const_cast<T*>(page) + int((keys - 1) & (g.page_size - 1)) * g.dim;
          for (int c = lane; c < g.dim; c += kWave) {
            kp[c] = fk[c];
            kp[c + g.kind_stride] = fv[c];
          }
        }
      }
      if (keys > int64_t(g.columns) * g.page_size) {
        w.l = NAN;  // a token past the table
      } else {
        w.keys(q, a.slabs, a.prefix_table, a.prefix_columns, 0, a.prefix, nullptr, nullptr, g, head, a.qscale);
        w.keys(q, a.slabs, table_row, g.columns, 0, keys, fk, fv, g, head, a.qscale);
      }
    }
    const float l = w.denominator();
    if (lane < g.dim) out[lane] = from_f32<DT>(finalize(w.acc[0], l));
    if (lane + kWave < g.dim) out[lane + kWave] = from_f32<DT>(finalize(w.acc[1], l));
  }
}

// ------------------------------------------------------------------- host ---
bool shared_shape(int b, int rows, int max_tokens, int h, int d, int page_size, int pps, int num_slabs, int prefix,
                  int columns, int layer, int layers, int dtype) {
  return b > 0 && b <= 65535 && rows > 0 && max_tokens > 0 && max_tokens <= rows && h > 0 && d > 0 && d <= 128 &&
         int64_t(b) * h <= 65535 && int64_t(rows) * h * d <= INT32_MAX && (page_size == 8 || page_size == 16 || page_size == 32) &&
         pps > 0 && num_slabs > 0 && int64_t(pps) * num_slabs <= INT32_MAX && prefix >= 0 && columns > 0 &&
         int64_t(b) * columns <= INT32_MAX && int64_t(columns) * page_size <= INT32_MAX &&
         int64_t(prefix) + int64_t(columns) * page_size <= INT32_MAX && layers > 0 && layer >= 0 && layer < layers &&
         dtype >= 0 && dtype <= 2;
}

hipError_t launch_shared(SharedArgs& a, int dtype) {
  const int64_t waves = int64_t(a.b) * a.max_tokens * a.g.heads;
  const int blocks = int(std::min<int64_t>((waves + 3) / 4, 1 << 20));
  if (dtype == kF32) shared_walk_kernel<kF32><<<blocks, 256>>>(a);
  else if (dtype == kF16) shared_walk_kernel<kF16><<<blocks, 256>>>(a);
  else shared_walk_kernel<kBF16><<<blocks, 256>>>(a);
  return hipGetLastError();
}

}  // namespace

extern "C" {

int mt_paged_append_slots(const void* k, const void* v, const uint64_t* slabs, const int64_t* slots, int rows, int h,
                          int d, int page_size, int pages_per_slab, int num_slabs, int layer, int layers, int dtype,
                          int kv_stride) {
  if (!k || !v || !slabs || !slots || rows < 1 || kv_stride < 0 ||
      !shared_shape(1, rows, 1, h, d, page_size, pages_per_slab, num_slabs, 0, 1, layer, layers, dtype))
    return hipErrorInvalidValue;
  const int64_t stride = kv_stride ? kv_stride : int64_t(h) * d;
  if (stride < int64_t(h) * d || rows * stride > INT32_MAX) return hipErrorInvalidValue;
  SlotArgs a{};
  a.k = k; a.v = v; a.slabs = slabs; a.slots = slots; a.stride = stride;
  a.g = make_geometry(h, d, page_size, pages_per_slab, num_slabs, 1, layer);
  const int esize = dtype == kF32 ? 4 : 2;
  const bool vec = (d * esize) % 16 == 0 && (stride * esize) % 16 == 0 && aligned16(k) && aligned16(v);
  a.units = int64_t(rows) * h * (vec ? d * esize / 16 : d);
  const int blocks = int(std::min<int64_t>((a.units + 255) / 256, 1 << 20));
#define MT_APPEND(DT)                                           \
  if (vec) append_slots_kernel<DT, true><<<blocks, 256>>>(a);   \
  else append_slots_kernel<DT, false><<<blocks, 256>>>(a);
  if (dtype == kF32) { MT_APPEND(kF32) }
  else if (dtype == kF16) { MT_APPEND(kF16) }
  else { MT_APPEND(kBF16) }
#undef MT_APPEND
  return hipGetLastError();
}

int mt_paged_shared_workspace_bytes(int rows, int b, int h, int d, int page_size, int prefix_tokens, int columns,
                                    int max_tokens, int dtype, size_t* bytes) {
  if (!bytes || !shared_shape(b, rows, max_tokens, h, d, page_size, 1, 1, prefix_tokens, columns, 0, 1, dtype))
    return hipErrorInvalidValue;
  *bytes = 0;
  return hipSuccess;
}

int mt_paged_shared_decode(void* out, const void* q, const void* k, const void* v, const uint64_t* slabs,
                           const int* prefix_table, const int* table, const int* offsets, int b, int h, int d,
                           int page_size, int pages_per_slab, int num_slabs, int prefix_tokens, int columns, int layer,
                           int layers, int dtype, int qkv_stride, void* workspace, size_t workspace_bytes) {
  if (!out || !q || !k || !v || !slabs || !table || !offsets || (prefix_tokens > 0 && !prefix_table) || qkv_stride < 0 ||
      !shared_shape(b, b, 1, h, d, page_size, pages_per_slab, num_slabs, prefix_tokens, columns, layer, layers, dtype))
    return hipErrorInvalidValue;
  const int64_t hd = int64_t(h) * d, stride = qkv_stride ? qkv_stride : hd;
  if (stride < hd || b * stride > INT32_MAX) return hipErrorInvalidValue;
  size_t need = 0;
  const int status = mt_paged_shared_workspace_bytes(b, b, h, d, page_size, prefix_tokens, columns, 1, dtype, &need);
  if (status) return status;
  if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return hipErrorInvalidValue;
  SharedArgs a{};
  a.out = out; a.q = q; a.k = k; a.v = v; a.slabs = slabs; a.prefix_table = prefix_table; a.table = table;
  a.lengths = offsets; a.b = b; a.rows = b; a.max_tokens = 1; a.prefix = prefix_tokens;
  a.prefix_columns = (prefix_tokens + page_size - 1) / page_size;
  a.qscale = (1.0f / std::sqrt(float(d))) * kLog2e;
  a.q_r = stride; a.o_r = hd;
  a.g = make_geometry(h, d, page_size, pages_per_slab, num_slabs, columns, layer);
  return launch_shared(a, dtype);
}

int mt_paged_shared_attention(void* out, const void* q, const uint64_t* slabs, const int* prefix_table,
                              const int* table, const int* lengths, const int* cu_tokens, int b, int rows,
                              int max_tokens, int h, int d, int page_size, int pages_per_slab, int num_slabs,
                              int prefix_tokens, int columns, int layer, int layers, int dtype, int q_stride,
                              int out_stride, void* workspace, size_t workspace_bytes) {
  if (!out || !q || !slabs || !table || !lengths || !cu_tokens || (prefix_tokens > 0 && !prefix_table) || q_stride < 0 ||
      out_stride < 0 ||
      !shared_shape(b, rows, max_tokens, h, d, page_size, pages_per_slab, num_slabs, prefix_tokens, columns, layer, layers,
                    dtype))
    return hipErrorInvalidValue;
  const int64_t hd = int64_t(h) * d, qs = q_stride ? q_stride : hd, os = out_stride ? out_stride : hd;
  if (qs < hd || os < hd || rows * qs > INT32_MAX || rows * os > INT32_MAX) return hipErrorInvalidValue;
  size_t need = 0;
  const int status =
      mt_paged_shared_workspace_bytes(rows, b, h, d, page_size, prefix_tokens, columns, max_tokens, dtype, &need);
  if (status) return status;
  if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return hipErrorInvalidValue;
  SharedArgs a{};
  a.out = out; a.q = q; a.slabs = slabs; a.prefix_table = prefix_table; a.table = table; a.lengths = lengths;
  a.cu_tokens = cu_tokens; a.b = b; a.rows = rows; a.max_tokens = max_tokens; a.prefix = prefix_tokens;
  a.prefix_columns = (prefix_tokens + page_size - 1) / page_size;
  a.qscale = (1.0f / std::sqrt(float(d))) * kLog2e;
  a.q_r = qs; a.o_r = os;
  a.g = make_geometry(h, d, page_size, pages_per_slab, num_slabs, columns, layer);
  return launch_shared(a, dtype);
}

}  // extern "C"
