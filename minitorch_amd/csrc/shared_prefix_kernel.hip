// Attention of a batch behind a shared prefix, and the K/V append through a slot
// map, for gfx950 (CDNA4, wave64). Pages, slabs and missing pages as in
// paged_attention_kernel.hip.
//
// Query i of request r: out = sum_j softmax_j(q k_j / sqrt(d)) v_j over the prefix's
// keys and the own keys 0 .. length + i. A piece of the keys leaves sum 2^(s - m) v,
// m and sum 2^(s - m) in fp32, and pieces join by their maxima, so that the prefix
// can be one piece of work for all requests and the own keys another. us in all
// (launches in a row): 64 requests x 12 heads of 64 fp16 behind 2048 tokens 16; 256 x
// 16 bf16 behind 16001 70; 512 x 25 bf16 behind 8192, own contexts up to 8192, 325 (5.4
// TB/s); 24 requests of up to 256 tokens x 16 heads of 128 bf16 behind 8100 360 (0.58
// PFLOP/s).
#include "mt_paged_device.h"
#include "../../include/mt_shared.h"
#include <algorithm>
#include <climits>

using namespace mt;

namespace {

// ---------------------------------------------------------------------------
// K/V rows to their pages through a slot map. VEC moves 16 bytes of K and of V per
// thread, neighbours side by side in the row and, for a head's columns, in the page. Bound
// by memory: 5001 rows of 25 heads of 64 in bf16 (64 MB moved) 11.6 us, 5.5 TB/s, as fast
// as a large copy; one launch's latency for few rows (64 rows of 12 heads 2.7 us).
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

// ---------------------------------------------------------------------------
// The fast path. A launch holds two kinds of work, whose results are partial:
// (accumulators, maximum, denominator) per query, head and piece of the keys,
// joined by merge_kernel.
//   * A prefix item attends a tile of 32 QT queries of one head -- of whatever
//     requests -- to a piece of the prefix, on the matrix cores: the piece is
//     read once for all of them.
//   * An own item attends a request's queries to its own pages: one query on the
//     VALU, streaming (decode), several on the matrix cores, causally.
// The first is bound by the matrix cores and the VALU between them, the second by
// memory, so that one launch that mixes them runs both at once.
constexpr int kPages = 512;  // pages of an item's keys, resolved into LDS
constexpr float kRescale = 6.f;
constexpr float kHalfShift = 9.f;  // 2^(kRescale + kHalfShift) is below fp16's largest

// Small pools' slab tables are copied to LDS while the first table entries are on
// their way, so that a page is one round trip away instead of two.
constexpr int kLdsSlabs = 512;

template <int NT>
struct SlabEntries {
  uint64_t entry[kLdsSlabs / NT];
  __device__ __forceinline__ void load(const SharedArgs& a) {
#pragma unroll
    for (int j = 0; j < kLdsSlabs / NT; ++j) {
      const int i = int(threadIdx.x) + j * NT;
      entry[j] = a.g.num_slabs <= kLdsSlabs && i < a.g.num_slabs ? a.slabs[i] : 0;
    }
  }
  __device__ __forceinline__ void store(uint64_t* s_slabs) const {
#pragma unroll
    for (int j = 0; j < kLdsSlabs / NT; ++j) s_slabs[threadIdx.x + j * NT] = entry[j];
  }
};
template <class T>
__device__ __forceinline__ const T* page_of(const SharedArgs& a, const uint64_t* s_slabs, int physical, int head) {
  if (!physical_in_pool(physical, a.g)) return nullptr;
  const int slab = slab_index(physical, a.g);
  return page_in_slab<T>(a.g.num_slabs <= kLdsSlabs ? s_slabs[slab] : a.slabs[slab], physical, a.g, head);
}

// How the launch is cut (made on the host). The prefix is units of prefix_unit keys;
// a (head, tile of 32 qt queries) has tile_units of them, all heads' tiles in a
// row, and a workgroup takes the next item_units: the same work for each, a piece
// of a tile or the end of one and the start of the next.
struct Plan {
  int waves;  // of a workgroup
  int qt, tiles, prefix_unit, tile_units, item_units;
  int pieces;  // most pieces a tile is cut into
  int64_t units, prefix_items;
  // own keys: splits of split_keys
  int split_keys, splits;
  // decode: waves per item and workgroups that take the rows of several splits
  int item_waves, more_blocks;
  // several queries: tiles of 32 own_qt queries; `listed` workgroups look up their items
  int own_qt, own_tiles;
  bool listed;
  int64_t own_blocks;
  float* partials;
};

// The first item that works on a tile (tile: head * tiles + tile), and how many do.
__device__ __forceinline__ int first_item(const Plan& p, int tile) {
  return int(unsigned(tile) * unsigned(p.tile_units) / unsigned(p.item_units));
}
__device__ __forceinline__ int pieces_of(const Plan& p, int tile) {
  return p.units ? int((unsigned(tile + 1) * unsigned(p.tile_units) - 1) / unsigned(p.item_units)) - first_item(p, tile) + 1 : 0;
}

// Elements of a query's partial: accumulators, maximum and denominator, 16-byte aligned.
template <int DP>
constexpr int part_row() { return DP + 4; }

template <int DP>
__device__ __forceinline__ float* part_of(const SharedArgs& a, const Plan& p, int piece, int head, int64_t row) {
  return p.partials + ((int64_t(piece) * a.g.heads + head) * a.rows + row) * part_row<DP>();
}

// Waves of a workgroup: four where their operands take 256 registers a lane, so
// that two workgroups still share a compute unit -- a prefix item and own ones
// (rows of 512 bytes stay with eight, for the sake of their rounds). Many rows of
// several queries take eight all the same: tiles of 128 queries of head dim 128 ask the
// caches for 32 KB every 4 MFLOP, more than they give (24 prompts behind 8100 tokens x
// 16 heads: 354 us with eight, 387 with four).
constexpr int shape_waves(int row_bytes, bool wide) { return row_bytes == 256 && !wide ? 4 : 8; }

// Staged keys of a workgroup: two halves of kHalf keys, K and V each. A wave takes
// blocks of 32 keys: with few waves per query group (KG <= kHalf / 32) a round is
// one half, staged while the other is computed; with more, both halves at once.
template <int DT, int DP, int WAVES>
struct Shape {
  static constexpr int ES = elem_bytes<DT>();
  static constexpr int EC = 16 / ES;          // elements per 16-byte chunk
  static constexpr int CPR = DP / EC;         // chunks per row
  static constexpr int RW = kWave / CPR;      // rows one load instruction of a wave fills
  static constexpr int kRowBytes = DP * ES;
  static constexpr int W = WAVES;
  static constexpr int NT = W * kWave;
  static constexpr int kHalf = kRowBytes == 128 ? 128 : 64;
  static constexpr int kBlocks = kHalf / 32;
  static constexpr int kPlane = kHalf * kRowBytes;
  static constexpr int NC = kHalf / (W * RW);  // loads per lane, K and V each
  static constexpr int DT32 = DP / 32;
  static constexpr int QW = DT == kF32 ? DP / 8 : DP / 16;  // 16-byte query registers
  static constexpr int OS = DP + 4;
  static constexpr size_t kMerge = size_t(W) * 32 * (OS + 2) * sizeof(float);
  static constexpr size_t kLds = size_t(4) * kPlane > kMerge ? size_t(4) * kPlane : kMerge;
  static constexpr int SW = kRowBytes == 128 ? 4 : 2;  // waves per SIMD: two workgroups a compute unit (512-byte rows: one)
  // Chunk p of key row r lies at chunk kpos / vpos of the row (both their own
  // inverse), so that the reads below are free of bank conflicts: K 16 bytes of
  // 32 consecutive rows, V 4 rows x 64 bytes (16-bit) or two rows 4 apart x 128
  // bytes (fp32).
  static __device__ __forceinline__ int kpos(int r, int p) { return CPR == 8 ? p ^ ((r >> 1) & 7) : p ^ (r & 15); }
  static __device__ __forceinline__ int vpos(int r, int p) {
    if constexpr (DT == kF32) return p ^ (((r >> 2) & 1) << 3);
    else return CPR == 8 ? p ^ (((r >> 1) & 1) << 2) : p ^ ((r & 3) << 2);
  }
};

// The largest of 16 scores (NaN ones are dropped), three a time in two chains; the
// compiler's own maxima also pass every product through a maximum with itself. Its
// first one stays: the compiler knows how long after the matrix product it may
// read the scores, and the instructions written here wait for its result.
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}
__device__ __forceinline__ float largest(const floatx16& s) {
  const float first = fmaxf(s[0], s[1]);
  float x = max3(first, s[2], s[3]), y = max3(first, s[4], s[5]);
  x = max3(x, s[6], s[7]);
  y = max3(y, s[8], s[9]);
  x = max3(x, s[10], s[11]);
  y = max3(y, s[12], s[13]);
  return max3(max3(x, s[14], s[15]), y, y);
}

// A tile of queries and the keys [k0, k1) of a table row that it attends (k0 a
// multiple of 32, at most kPages pages): query j those up to limit + j.
struct Tile {
  const void* q;  // row of query 0, at the head's columns
  int nq, qt;
  const int* table_row;
  int columns, k0, k1;
  int64_t limit;
  float* part;  // partial of query 0 (the others follow)
};

// S^T = K Q^T in 32x32 MFMAs (keys x queries: two lanes share a query and hold
// half of a block's scores of it each), online softmax in registers, O^T += V^T
// P^T with the scores' own layout as the B operand. For 16-bit types P is split
// into a high and a low part of the type (two MFMAs), so that the weights keep 16
// (bf16) or 22 (fp16) bits and the output is as exact as the other attention
// kernels'; fp16's are taken 2^kHalfShift larger, whose low parts would
// otherwise end at 2^-24. The exponentials' reference moves when a score exceeds
// it by kRescale only.
template <int DT, int DP, int W, Rows FULL>
__device__ __forceinline__ void attend_tile(const SharedArgs& a, const Tile& t, int head, char* s_raw,
                                            typename Elem<DT>::T const** s_page, uint64_t* s_slabs, int* s_missing) {
  using T = typename Elem<DT>::T;
  using S = Shape<DT, DP, W>;
  constexpr int EC = S::EC, CPR = S::CPR, NC = S::NC, DT32 = S::DT32, QW = S::QW, NT = S::NT;
  constexpr float kShift = DT == kF16 ? kHalfShift : 0.f;
  constexpr int CH = DP == 64 ? 4 : 2;  // chains of an fp32 block's sums
  const Geometry& g = a.g;
  const int dim = FULL == kRowsFull ? DP : g.dim, chunks = dim / EC;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // keeps this tile's terms out of the registers of the tiles before
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qt_n = t.qt, kg_n = W / qt_n;
  const int kg = wave / qt_n, qt = wave - kg * qt_n;
  const int grp = lane >> 5, col = lane & 31;
  const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)s_raw));

  // B operand of S^T: chunks 2 s + grp of the lane's query. Products with nothing but
  // padding are left out for fp32 rows of up to 64, whose products are slow (110 requests
  // x 25 heads of 32 behind 6697 tokens: 55 us instead of 74); elsewhere the branches cost
  // more than they save (10 x 5 tokens x 12 heads of 72 in fp16 behind 1272: 19.3 and 17.6).
  constexpr bool TRIM = DT == kF32 && DP == 64 && FULL == kRowsPadded;
  const int s_end = (chunks + 1) / 2, d_end = (dim + 31) / 32;
  auto in_s = [&](int s) { return !TRIM || s < s_end; };
  auto in_d = [&](int d) { return !TRIM || d < d_end; };
  const int q0 = qt * 32, qi = q0 + col;
  const bool live = q0 < t.nq;
  const T* qrow = static_cast<const T*>(t.q) + (qi < t.nq ? qi : 0) * a.q_r;
  u32x4 qv[QW];
#pragma unroll
  for (int s = 0; s < QW; ++s) {
    const int p = 2 * s + grp;
    qv[s] = *global_view(reinterpret_cast<const u32x4*>(p < chunks ? qrow + p * EC : reinterpret_cast<const T*>(g_fill + 4)));
  }

  // the pages of the keys
  const int pages = (t.k1 - t.k0 + g.page_size - 1) >> g.log2_page;
  int physical[kPages / NT];
#pragma unroll
  for (int j = 0; j < kPages / NT; ++j) {
    const int i = tid + j * NT, column = (t.k0 >> g.log2_page) + i;
    physical[j] = i < pages && column < t.columns ? t.table_row[column] : -1;
  }
  SlabEntries<NT> slabs;
  slabs.load(a);
  if (tid == 0) *s_missing = 0;
  slabs.store(s_slabs);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPages / NT; ++j) {
    const int i = tid + j * NT;
    if (i >= pages) break;
    const T* page = page_of<T>(a, s_slabs, physical[j], head);
    s_page[i] = page;
    if (!page) *s_missing = 1;
  }
  __syncthreads();
  const bool plain = FULL == kRowsFull && !*s_missing;

  // Keys [k, k + kHalf) into half `h`. Keys past the end are zero; a missing
  // page is NaN in K (its scores are NaN) and zero in V.
  const int sr = wave * S::RW + lane / CPR, spos = lane % CPR;
  auto stage = [&](int k, int h) {
    const uint32_t lk = lds0 + h * 2 * S::kPlane + wave * 1024, lv = lk + S::kPlane;
    if (plain && k + S::kHalf <= t.k1) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int r = sr + n * W * S::RW;
        const T* page = s_page[(k + r - t.k0) >> g.log2_page] + (r & (g.page_size - 1)) * dim;
        stage16(page + S::kpos(r, spos) * EC, lk + n * W * 1024);
        stage16(page + g.kind_stride + S::vpos(r, spos) * EC, lv + n * W * 1024);
      }
    } else {
      int row = sr;
      asm volatile("" : "+v"(row));  // keeps this rarer path's terms out of the registers of the loop
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int r = row + n * W * S::RW, key = k + r;
        // a block wholly past the keys is never read
        if (k + ((wave * S::RW + n * W * S::RW) & ~31) >= t.k1) continue;
        const int pk = S::kpos(r, spos), pv = S::vpos(r, spos);
        const T* kp = reinterpret_cast<const T*>(g_fill + 4);
        const T* vp = kp;
        if (key < t.k1) {
          const T* page = s_page[(key - t.k0) >> g.log2_page];
          if (!page) {
            kp = reinterpret_cast<const T*>(g_fill);
          } else {
            page += (r & (g.page_size - 1)) * dim;
            if (pk < chunks) kp = page + pk * EC;
            if (pv < chunks) vp = page + g.kind_stride + pv * EC;
          }
        }
        stage16(kp, lk + n * W * 1024);
        stage16(vp, lv + n * W * 1024);
      }
    }
  };

  float m = -INFINITY, l = 0.f;
  const float unscale = 1.f / a.qscale;
  float threshold = -INFINITY;  // a product past it moves the reference
  floatx16 o[DT32];
#pragma unroll
  for (int d = 0; d < DT32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  const int64_t own_limit = t.limit + qi;
  const int last_key = int(own_limit < t.k1 ? own_limit : t.k1 - 1);  // of this lane's query

  // A score past the reference by kRescale moves it. (Each lane asks for its own
  // half of the keys; a query's first ones, m = -inf, move it too.)
  auto refer = [&](float mine) {
    if (__any(mine > threshold)) {
      const float mn = fmaxf(m, max_halves(mine) * a.qscale);
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
      m = mn;
      threshold = (m + kRescale) * unscale;
    }
    return m == -INFINITY ? 0.f : m - kShift;
  };
  // The scores' weights, added to the denominator.
  auto weigh = [&](floatx16& sc, float ref) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = fast_exp2(fmaf(sc[i], a.qscale, -ref));
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = sc[i] + sc[i + 8];
#pragma unroll
    for (int w = 4; w > 0; w /= 2)
#pragma unroll
      for (int i = 0; i < w; ++i) sum[i] += sum[i + w];
    l += sum[0];
  };
  // K's operand s of the block of 32 keys at s_k, for S^T.
  auto read_k = [&](const T* s_k, int s) {
    const int p = 2 * s + grp;
    return *reinterpret_cast<const u32x4*>(s_k + col * DP + S::kpos(col, p) * EC);
  };
  // O^T += V^T P^T for 16-bit types, 16 keys a step: slot j < 4 of a lane holds key
  // 16 s + 4 grp + j, slot j >= 4 key 16 s + 8 + 4 grp + j - 4, in P as in V^T.
  auto accumulate = [&](const T* s_v, const floatx16& sc) {
    const int t16 = lane & 15;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 hi, lo;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t h2, l2;
        SplitP<DT == kF32 ? kF16 : DT>::split(sc[8 * s + 2 * w], sc[8 * s + 2 * w + 1], h2, l2);
        hi[w] = h2;
        lo[w] = l2;
      }
      u32x4 vt[DT32];
#pragma unroll
      for (int d = 0; d < DT32; ++d) {
        if (!in_d(d)) break;
        const int rr = 4 * grp + (t16 >> 2);
        const int p = 4 * d + ((lane >> 4) & 1) * 2 + ((t16 & 3) >> 1);
        const T* v_at = s_v + (16 * s + rr) * DP + S::vpos(rr, p) * 8 + (t16 & 1) * 4;
        const uint2 x = read_transposed(v_at), y = read_transposed(v_at + 8 * DP);
        vt[d] = u32x4{x.x, x.y, y.x, y.y};
      }
      // (no product waits for the one before it)
#pragma unroll
      for (int d = 0; d < DT32; ++d)
        if (in_d(d)) o[d] = mfma32<DT>(vt[d], hi, o[d]);
#pragma unroll
      for (int d = 0; d < DT32; ++d)
        if (in_d(d)) o[d] = mfma32<DT>(vt[d], lo, o[d]);
    }
  };
  auto keys_at = [&](int h, int at) { return reinterpret_cast<const T*>(s_raw + h * 2 * S::kPlane) + at * DP; };

  // One block of 32 keys from `base` on, at row `at` of half h: lane holds the scores of
  // keys base + 8 (i / 4) + 4 grp + i % 4 of query qi.
  auto block = [&](int base, int h, int at) {
    const T* const s_k = keys_at(h, at);
    const T* const s_v = s_k + S::kPlane / S::ES;
    floatx16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
    if constexpr (DT == kF32) {
      // short chains of sums
      floatx16 part[CH];
#pragma unroll
      for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) part[j][i] = 0.f;
#pragma unroll
      for (int s = 0; s < QW; ++s) {
        if (!in_s(s)) break;
        const u32x4 kf = read_k(s_k, s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          floatx16& c = part[j % CH];
          c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[j]), __uint_as_float(qv[s][j]), c, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = (part[0][i] + part[1][i]) + (CH == 4 ? part[CH - 2][i] + part[CH - 1][i] : 0.f);
    } else {
#pragma unroll
      for (int s = 0; s < QW; ++s)
        if (in_s(s)) sc = mfma32<DT>(read_k(s_k, s), qv[s], sc);
    }
    // limits, only for blocks that reach past one (a wave-uniform test)
    if (base + 31 > t.limit + q0 || base + 32 > t.k1) {
      const int last = last_key - base - 4 * grp;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x = 8 * (i >> 2) + (i & 3) > last ? -INFINITY : sc[i];
        asm volatile("" : "+v"(x));  // keeps this a branch: 46 instructions of a block's 190 without it
        sc[i] = x;
      }
    }
    weigh(sc, refer(largest(sc)));
    if constexpr (DT == kF32) {
      // a block's sums start at zero, in chains, and are added to the running ones
#pragma unroll
      for (int d = 0; d < DT32; ++d) {
        if (!in_d(d)) break;
        floatx16 ob[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
          for (int i = 0; i < 16; ++i) ob[j][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int rr = 8 * (i >> 2) + 4 * grp + (i & 3), dd = 32 * d + col;
          const float vv = s_v[rr * DP + S::vpos(rr, dd >> 2) * 4 + (dd & 3)];
          ob[i % CH] = __builtin_amdgcn_mfma_f32_32x32x2f32(vv, sc[i], ob[i % CH], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          o[d][i] += (ob[0][i] + ob[1][i]) + (CH == 4 ? ob[CH - 2][i] + ob[CH - 1][i] : 0.f);
      }
    } else {
      accumulate(s_v, sc);
    }
  };
  // Two blocks, both whole and within the limits, at rows at0 and at1 (16-bit types,
  // where a lane has registers for it): their products take turns, and the reference is
  // looked at once.
  auto two_blocks = [&](int h, int at0, int at1) {
    const T *const k0 = keys_at(h, at0), *const k1 = keys_at(h, at1);
    floatx16 s0, s1;
#pragma unroll
    for (int i = 0; i < 16; ++i) s0[i] = s1[i] = 0.f;
#pragma unroll
    for (int s = 0; s < QW; ++s) {
      if (!in_s(s)) break;
      s0 = mfma32<DT>(read_k(k0, s), qv[s], s0);
      s1 = mfma32<DT>(read_k(k1, s), qv[s], s1);
    }
    const float ref = refer(fmaxf(largest(s0), largest(s1)));
    weigh(s0, ref);
    weigh(s1, ref);
    accumulate(k0 + S::kPlane / S::ES, s0);
    accumulate(k1 + S::kPlane / S::ES, s1);
  };

  const bool both = kg_n > S::kBlocks;  // rounds of both halves
  stage(t.k0, 0);
  if (both && t.k0 + S::kHalf < t.k1) stage(t.k0 + S::kHalf, 1);
#pragma unroll
  for (int s = 0; s < QW; ++s) asm volatile("" : "+v"(qv[s]));  // the query has arrived before the loop
  if (both) {
    const int h = kg / S::kBlocks, at = (kg - h * S::kBlocks) * 32;
    for (int k = t.k0; k < t.k1; k += 2 * S::kHalf) {
      wait_staged<0>();
      __syncthreads();
      const int base = k + h * S::kHalf + at;
      if (live && h < 2 && base < t.k1 && base <= t.limit + min(q0 + 31, t.nq - 1)) block(base, h, at);
      const int next = k + 2 * S::kHalf;
      if (next < t.k1) {
        __syncthreads();
        stage(next, 0);
        if (next + S::kHalf < t.k1) stage(next + S::kHalf, 1);
      }
    }
  } else {
    int h = 0;
    for (int k = t.k0; k < t.k1; k += S::kHalf, h ^= 1) {
      wait_staged<0>();
      __syncthreads();  // the half's keys are there, and the half before is done with
      if (k + S::kHalf < t.k1) stage(k + S::kHalf, h ^ 1);
      if (live) {
        const int step = kg_n * 32;
        int at = kg * 32;
        if constexpr (DT != kF32 && S::SW == 2)
          for (; at + step < S::kHalf; at += 2 * step) {
            const int past = k + at + step + 32;
            if (past > t.k1 || past - 1 > t.limit + q0) break;
            two_blocks(h, at, at + step);
          }
        for (; at < S::kHalf; at += step) {
          const int base = k + at;
          if (base >= t.k1 || base > t.limit + min(q0 + 31, t.nq - 1)) break;
          block(base, h, at);
        }
      }
    }
  }

  // The waves that share queries meet in LDS; then every thread joins four dims
  // of a query. O^T lane layout: dims 32 d + 8 (i / 4) + 4 grp + i % 4 of query qi.
  l = add_halves(l);
  m -= kShift;
  constexpr int R = part_row<DP>();
  if (kg_n == 1) {
    if (qi < t.nq) {
      float* row = t.part + qi * R;
#pragma unroll
      for (int d = 0; d < DT32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(row + 32 * d + 2 * i + 4 * grp) = float4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
      if (grp == 0) *reinterpret_cast<float2*>(row + DP) = float2{m, l};
    }
    return;
  }
  float* const s_o = reinterpret_cast<float*>(s_raw);
  float2* const s_ml = reinterpret_cast<float2*>(s_o + W * 32 * S::OS);
  const int tq = 32 * qt_n;
  __syncthreads();
  {
    float* row = s_o + (kg * tq + qi) * S::OS + 4 * grp;
#pragma unroll
    for (int d = 0; d < DT32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(row + 32 * d + 2 * i) = float4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
    if (grp == 0) s_ml[kg * tq + qi] = float2{m, l};
  }
  __syncthreads();
  for (int u = tid; u < t.nq * (DP / 4); u += NT) {
    const int q = u / (DP / 4), dd = 4 * (u - q * (DP / 4));
    float M = -INFINITY, L = 0.f;
    for (int k = 0; k < kg_n; ++k) M = fmaxf(M, s_ml[k * tq + q].x);
    float4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < kg_n; ++k) {
      const float2 ml = s_ml[k * tq + q];
      const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
      const float4 x = *reinterpret_cast<const float4*>(s_o + (k * tq + q) * S::OS + dd);
      L = fmaf(ml.y, w, L);  // a NaN denominator (missing page) stays
      if (isnan(ml.y)) L = NAN;
      acc.x = fmaf(x.x, w, acc.x); acc.y = fmaf(x.y, w, acc.y);
      acc.z = fmaf(x.z, w, acc.z); acc.w = fmaf(x.w, w, acc.w);
    }
    *reinterpret_cast<float4*>(t.part + q * R + dd) = acc;
    if (dd == 0) *reinterpret_cast<float2*>(t.part + q * R + DP) = float2{M, L};
  }
}

// Own keys of one query (decode), streamed: a wave covers 8 tokens a step, eight
// lanes a token, U steps in flight; item_waves waves share an item. The keys of
// split `split` of row `row`, or with split -1 those of a row that is one split;
// the last split appends and scores the new token.
// All threads of the workgroup enter (barriers); `on` where the group has an item.
// What does not depend on the row's length -- table entries, query, new token --
// is loaded with it, in one round trip.
template <int DT, int DP, int WAVES, Rows FULL>
__device__ __forceinline__ void stream_item(const SharedArgs& a, const Plan& p, bool on, int row, int head, int split,
                                            float* s_state, uint64_t* s_slabs, bool& slabs_there) {
  using T = typename Elem<DT>::T;
  constexpr int G = 8, DL = DP / G, RB = kWave / G;
  constexpr int U = DL * elem_bytes<DT>() >= 64 ? 1 : DL * elem_bytes<DT>() >= 32 ? 2 : 4;
  using C = Chunk<DT, DL, FULL, G>;
  const Geometry& g = a.g;
  const int dim = FULL == kRowsFull ? DP : g.dim;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & (kWave - 1);
  const int W = p.item_waves, gw = wave % W, first_wave = wave - gw;
  const int col0 = C::first_col(lane % G), tok = lane / G;
  // before the prefix items' waves, whose products leave these few turns to ask for more keys
  // (256 requests x 16 heads behind 16001 tokens: 74.6 us with it, 84.5 without)
  __builtin_amdgcn_s_setprio(2);
  const bool whole = split < 0;
  split = max(split, 0);
  const int t0 = split * p.split_keys;
  const int rel0 = (gw + W * lane) * RB;  // lane i: this wave's step i
  const int* const table_row = a.table + int64_t(row) * g.columns;
  const int64_t qrow = int64_t(row) * a.q_r + int64_t(head) * dim;
  const int64_t column0 = (int64_t(t0) + rel0) >> g.log2_page;
  int physical = -1, offset = -1;
  Query<DT, DP, FULL, G> qv;
  C kn, vn;
  if (on) {
    offset = a.lengths[row];
    if (rel0 < p.split_keys && column0 < g.columns) physical = table_row[column0];
    qv.load(static_cast<const T*>(a.q) + qrow, col0, dim, a.qscale);
    if (gw == 0) {
      kn.load(static_cast<const T*>(a.k) + qrow + col0, col0, dim);
      vn.load(static_cast<const T*>(a.v) + qrow + col0, col0, dim);
    }
  }
  if (!slabs_there) {
    SlabEntries<WAVES * kWave> slabs;
    slabs.load(a);
    slabs.store(s_slabs);
    __syncthreads();
    slabs_there = true;
  }
  const int64_t L = int64_t(offset) + 1;
  on = offset >= 0 && L <= int64_t(g.columns) * g.page_size;
  const int nsplit = on ? int((uint32_t(L) + uint32_t(p.split_keys) - 1) / uint32_t(p.split_keys)) : 0;
  on = whole ? nsplit == 1 : split < nsplit;
  Softmax<DL, G> st;
  st.init();
  if (on) {
    const int t1 = int(L < int64_t(t0) + p.split_keys ? L : int64_t(t0) + p.split_keys);
    const bool owns_new = split == nsplit - 1;
    const int ntok = (owns_new ? t1 - 1 : t1) - t0;
    const int new_physical = owns_new && gw == 0 ? table_row[(t1 - 1) >> g.log2_page] : -1;
    const T* page = rel0 < ntok ? page_of<T>(a, s_slabs, physical, head) : nullptr;
    const uint64_t at = reinterpret_cast<uintptr_t>(page);
    const int at_lo = int(uint32_t(at)), at_hi = int(uint32_t(at >> 32));
    const int steps_all = (ntok + RB - 1) / RB;
    const int steps = steps_all > gw ? (steps_all - gw + W - 1) / W : 0;
    for (int i0 = 0; i0 < steps; i0 += U) {
      C kc[U], vc[U];
      bool valid[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u, kWave - 1);
        const int rel = (gw + W * (i0 + u)) * RB + tok;
        valid[u] = rel < ntok;
        const T* base = reinterpret_cast<const T*>(uint64_t(uint32_t(__builtin_amdgcn_readlane(at_hi, i))) << 32 |
                                                   uint32_t(__builtin_amdgcn_readlane(at_lo, i)));
        if (valid[u] && base) {
          const T* kp = base + ((t0 + rel) & (g.page_size - 1)) * dim + col0;
          kc[u].template load<true>(kp, col0, dim);
          vc[u].template load<true>(kp + g.kind_stride, col0, dim);
        } else {
          kc[u].nan_fill();
          vc[u].nan_fill();
        }
      }
      float s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) s[u] = qv.score(kc[u]);
      // one move of the running maximum for the U tokens; no scores but -Inf leave it
      float top = st.m;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (valid[u]) top = fmaxf(top, s[u]);
      const float ref = top == -INFINITY ? 0.f : top;
      const float alpha = fast_exp2(st.m - ref);
      st.l *= alpha;
#pragma unroll
      for (int e = 0; e < DL; ++e) st.acc[e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!valid[u]) continue;
        const float w = fast_exp2(s[u] - ref);
        float vf[DL];
        vc[u].to_float(vf);
        st.l += w;
#pragma unroll
        for (int e = 0; e < DL; ++e) st.acc[e] = fmaf(w, vf[e], st.acc[e]);
      }
      st.m = top;
    }
    if (owns_new && gw == 0) {
      // the new token, by the first eight lanes: written to its page and scored
      const T* np = page_of<T>(a, s_slabs, new_physical, head);
      if (np && lane < G) {
        T* kp = const_cast<T*>(np) + ((t1 - 1) & (g.page_size - 1)) * dim + col0;
        T* vp = kp + g.kind_stride;
#pragma unroll
        for (int i = 0; i < C::NV; ++i) {
          if (FULL == kRowsPadded && col0 + i * G * per16<DT>() >= dim) break;
          global_view(reinterpret_cast<u32x4*>(kp))[i * G] = kn.raw[i];
          global_view(reinterpret_cast<u32x4*>(vp))[i * G] = vn.raw[i];
        }
      }
      if (!np) { kn.nan_fill(); vn.nan_fill(); }
      const float sc = qv.score(kn);
      if (lane < G) {
        float vf[DL];
        vn.to_float(vf);
        const float top = fmaxf(st.m, sc), ref = top == -INFINITY ? 0.f : top;
        const float alpha = fast_exp2(st.m - ref), w = fast_exp2(sc - ref);
        st.l = fmaf(st.l, alpha, w);
#pragma unroll
        for (int e = 0; e < DL; ++e) st.acc[e] = fmaf(w, vf[e], st.acc[e] * alpha);
        st.m = top;
      }
    }
  }
  // States of the 16-lane rows by DPP, then the item's 4 W of them in LDS.
  float* const s_acc = s_state;  // [4 WAVES][DP]
  float2* const s_ml = reinterpret_cast<float2*>(s_state + 4 * WAVES * DP);
  st.row_merge();
  if ((lane & 15) < G) {
    const int si = wave * 4 + (lane >> 4);
#pragma unroll
    for (int i = 0; i < DL; ++i) s_acc[si * DP + col0 + C::col_of(i)] = st.acc[i];
    if ((lane & 15) == 0) s_ml[si] = float2{st.m, st.l};
  }
  __syncthreads();
  if (on) {
    float* part = part_of<DP>(a, p, p.pieces + split, head, row);
    for (int d = gw * kWave + lane; d < DP; d += W * kWave) {
      float M = -INFINITY, L = 0.f, acc = 0.f;
      for (int j = first_wave * 4; j < (first_wave + W) * 4; ++j) M = fmaxf(M, s_ml[j].x);
      for (int j = first_wave * 4; j < (first_wave + W) * 4; ++j) {
        const float2 ml = s_ml[j];
        const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
        L = fmaf(ml.y, w, L);
        if (isnan(ml.y)) L = NAN;  // also where no score was a number
        acc = fmaf(s_acc[j * DP + d], w, acc);
      }
      part[d] = acc;
      if (d == 0) { part[DP] = M; part[DP + 1] = L; }
    }
  }
  __syncthreads();
}

// The rows of several splits: every workgroup counts them (rows in chunks of a thread
// each) and takes its share. They start before the other rows, which are short
// then, so that none is left alone at the end.
template <int DT, int DP, int WAVES, Rows FULL>
__device__ __forceinline__ void stream_more(const SharedArgs& a, const Plan& p, int block, float* s_state, uint64_t* s_slabs,
                                            int* s_count) {
  constexpr int NT = WAVES * kWave;
  const Geometry& g = a.g;
  const int tid = threadIdx.x, groups = WAVES / p.item_waves, group = (tid >> 6) / p.item_waves;
  const int64_t cap = int64_t(g.columns) * g.page_size;
  bool slabs_there = false;
  int64_t set = block;  // this workgroup's next set of `groups` items, less those of the chunks before
  for (int r0 = 0; r0 < a.b; r0 += NT) {
    int more = 0;
    if (r0 + tid < a.b) {
      const int64_t L = int64_t(a.lengths[r0 + tid]) + 1;
      if (L > p.split_keys && L <= cap) more = int((L - 1) / p.split_keys) + 1;
    }
    // inclusive sums over the chunk
    int sum = wave_inclusive_add(more);
    __syncthreads();
    if ((tid & 63) == 63) s_count[NT + (tid >> 6)] = sum;
    __syncthreads();
    for (int w = 0; w < (tid >> 6); ++w) sum += s_count[NT + w];
    s_count[tid] = sum;
    __syncthreads();
    const int64_t items = int64_t(s_count[NT - 1]) * g.heads;
    const int64_t sets = (items + groups - 1) / groups;
    for (; set < sets; set += p.more_blocks) {
      const int64_t item = set * groups + group;
      const bool on = item < items;
      const int x = on ? int(item / g.heads) : 0, head = on ? int(item - int64_t(x) * g.heads) : 0;
      int i = 0;  // the first row whose sum passes x
#pragma unroll
      for (int step = NT / 2; step > 0; step >>= 1)
        if (s_count[i + step - 1] <= x) i += step;
      const int before = i ? s_count[i - 1] : 0;
      stream_item<DT, DP, WAVES, FULL>(a, p, on, on ? r0 + i : 0, head, x - before, s_state, s_slabs, slabs_there);
    }
    set -= sets;
  }
}

// Own keys of several queries: an item is a tile of a request's queries, one of its
// splits and a head. The host knows bounds only: each request as long as the longest,
// each context as long as the table. Up to eight rounds of such workgroups
// that is as fast as counting (96 requests of one token and 32 prompts of 16-512, 12
// heads, table of 1024: 118 us, counted 121); where the bounds give more, eight
// rounds count the items that there are (kListed requests at once) and share them out: 500
// requests of one token and 12 prompts of 500-2048 behind 2048 tokens, 12 heads, table of
// 8192: 366 us, with a workgroup for each of 245000 bounds 1250.
constexpr int kListed = 256;

template <int DT, int DP, int W, Rows FULL>
__device__ __forceinline__ void own_item(const SharedArgs& a, const Plan& p, int r, const Request& rq, int tile, int split,
                                         int head, char* s_raw, typename Elem<DT>::T const** s_page, uint64_t* s_slabs,
                                         int* s_missing) {
  using T = typename Elem<DT>::T;
  const Geometry& g = a.g;
  const int q0 = tile * 32 * p.own_qt;
  if (rq.length < 0 || q0 >= rq.tokens) return;
  Tile t;
  t.nq = min(32 * p.own_qt, rq.tokens - q0);
  // a key past the table is a missing page: one of them is enough
  const int64_t end = min(int64_t(rq.length) + q0 + t.nq, int64_t(g.columns) * g.page_size + 1);
  const int64_t k0 = int64_t(split) * p.split_keys;
  if (k0 >= end) return;
  const int64_t row = int64_t(rq.row0) + q0;
  t.q = static_cast<const T*>(a.q) + row * a.q_r + int64_t(head) * g.dim;
  t.qt = p.own_qt;
  while (t.qt > 1 && 16 * t.qt >= t.nq) t.qt /= 2;  // few queries leave more waves to their keys
  t.table_row = a.table + int64_t(r) * g.columns;
  t.columns = g.columns;
  t.k0 = int(k0);
  t.k1 = int(min(end, k0 + p.split_keys));
  t.limit = int64_t(rq.length) + q0;
  t.part = part_of<DP>(a, p, p.pieces + split, head, row);
  attend_tile<DT, DP, W, FULL>(a, t, head, s_raw, s_page, s_slabs, s_missing);
}

template <int DT, int DP, int W, Rows FULL>
__device__ __forceinline__ void listed_items(const SharedArgs& a, const Plan& p, int block, char* s_raw,
                                             typename Elem<DT>::T const** s_page, uint64_t* s_slabs, int* s_missing,
                                             int* s_count) {
  const Geometry& g = a.g;
  const int tid = threadIdx.x, tq = 32 * p.own_qt;
  const int64_t cap = int64_t(g.columns) * g.page_size;
  int64_t next = block;  // this workgroup's next item, less those of the requests before
#pragma unroll 1
  for (int r0 = 0; r0 < a.b; r0 += kListed) {
    // tiles times splits of the last of them (an early tile's later splits are none)
    int items = 0;
    if (tid < kListed && r0 + tid < a.b) {
      const Request rq = request_of(a, r0 + tid);
      if (rq.length >= 0 && rq.tokens > 0) {
        const int64_t end = min(int64_t(rq.length) + rq.tokens, cap + 1);
        items = (rq.tokens + tq - 1) / tq * int((end + p.split_keys - 1) / p.split_keys);
      }
    }
    int sum = wave_inclusive_add(items);
    __syncthreads();  // the requests before are done with
    if (tid < kListed && (tid & 63) == 63) s_count[kListed + (tid >> 6)] = sum;
    __syncthreads();
    if (tid < kListed) {
      for (int w = 0; w < (tid >> 6); ++w) sum += s_count[kListed + w];
      s_count[tid] = sum;
    }
    __syncthreads();
    const int64_t all = int64_t(s_count[kListed - 1]) * g.heads;
#pragma unroll 1
    for (; next < all; next += p.own_blocks) {
      const int x = __builtin_amdgcn_readfirstlane(int(next / g.heads));
      const int head = __builtin_amdgcn_readfirstlane(int(next - int64_t(x) * g.heads));
      int i = 0;  // the first request whose sum passes x
#pragma unroll
      for (int step = kListed / 2; step > 0; step >>= 1)
        if (s_count[i + step - 1] <= x) i += step;
      i = __builtin_amdgcn_readfirstlane(i);
      const int item = x - (i ? __builtin_amdgcn_readfirstlane(s_count[i - 1]) : 0);
      const Request rq = request_of(a, r0 + i);
      const int tiles = max(1, (rq.tokens + tq - 1) / tq), split = item / tiles;
      own_item<DT, DP, W, FULL>(a, p, r0 + i, rq, item - split * tiles, split, head, s_raw, s_page, s_slabs, s_missing);
      __syncthreads();  // the LDS is done with
    }
    next -= all;
  }
}

// Own: one new token per request; several, a workgroup per item; several, shared out.
enum Own { kOwnToken, kOwnTiles, kOwnListed };

template <int DT, int DP, int W, Rows FULL, Own OWN>
__global__ __launch_bounds__((Shape<DT, DP, W>::NT)) __attribute__((amdgpu_waves_per_eu((Shape<DT, DP, W>::SW))))
void shared_kernel(SharedArgs a, Plan p) {
  using T = typename Elem<DT>::T;
  using S = Shape<DT, DP, W>;
  __shared__ const T* s_page[kPages];
  __shared__ uint64_t s_slabs[kLdsSlabs];
  __shared__ int s_missing;
  __shared__ __align__(16) char s_raw[S::kLds];
  const Geometry& g = a.g;
  // The prefix items first: they are the long ones, one a compute unit where own
  // items follow, which then take the rest of it. Neighbours go to one XCD (the
  // workgroups of a launch are dealt to the eight in turn), so that the tiles of a
  // head share its keys in that XCD's L2.
  int index = int(blockIdx.x);
  if (index < p.prefix_items) {
    const int whole = int(p.prefix_items) & ~7;
    if (index < whole) index = (index & 7) * (whole >> 3) + (index >> 3);
    const int end = int(min(p.units, int64_t(index + 1) * p.item_units));
#pragma unroll 1
    for (int at = index * p.item_units; at < end;) {
      const int head_tile = __builtin_amdgcn_readfirstlane(int(unsigned(at) / unsigned(p.tile_units)));
      const int unit = at - head_tile * p.tile_units, n = min(p.tile_units - unit, end - at);
      const int head = __builtin_amdgcn_readfirstlane(int(unsigned(head_tile) / unsigned(p.tiles)));
      const int tile = head_tile - head * p.tiles;
      const int64_t row = int64_t(tile) * 32 * p.qt;
      Tile t;
      t.q = static_cast<const T*>(a.q) + row * a.q_r + int64_t(head) * g.dim;
      t.nq = int(min(int64_t(32 * p.qt), a.rows - row));
      t.qt = p.qt;
      t.table_row = a.prefix_table;
      t.columns = a.prefix_columns;
      t.k0 = unit * p.prefix_unit;
      t.k1 = min(a.prefix, (unit + n) * p.prefix_unit);
      t.limit = INT_MAX;
      t.part = part_of<DP>(a, p, index - __builtin_amdgcn_readfirstlane(first_item(p, head_tile)), head, row);
      attend_tile<DT, DP, W, FULL>(a, t, head, s_raw, s_page, s_slabs, &s_missing);
      at += n;
      if (at < end) __syncthreads();  // the LDS is done with
    }
    return;
  }
  index -= int(p.prefix_items);
  if constexpr (OWN == kOwnToken) {
    if (index < p.more_blocks) {
      stream_more<DT, DP, W, FULL>(a, p, index, reinterpret_cast<float*>(s_raw), s_slabs, reinterpret_cast<int*>(s_page));
      return;
    }
    index -= p.more_blocks;
    const int groups = S::W / p.item_waves;
    const int64_t item = int64_t(index) * groups + (threadIdx.x >> 6) / p.item_waves;
    const bool on = item < int64_t(a.b) * g.heads;
    const int row = on ? int(item / g.heads) : 0;
    bool slabs_there = false;
    stream_item<DT, DP, W, FULL>(a, p, on, row, on ? int(item - int64_t(row) * g.heads) : 0, -1,
                              reinterpret_cast<float*>(s_raw), s_slabs, slabs_there);
  } else if constexpr (OWN == kOwnTiles) {
    // (split, tile, request, head), the last tiles, which attend the most keys, first (16
    // prompts of 453 x 16 heads fp32: 171 us, 204 in order)
    const int i = index / g.heads, head = index - i * g.heads;
    const int st = i / a.b, r = i - st * a.b;
    const int split = st / p.own_tiles, tile = p.own_tiles - 1 - (st - split * p.own_tiles);
    own_item<DT, DP, W, FULL>(a, p, r, request_of(a, r), tile, split, head, s_raw, s_page, s_slabs, &s_missing);
  } else {
    __shared__ int s_count[kListed + kListed / kWave];
    listed_items<DT, DP, W, FULL>(a, p, index, s_raw, s_page, s_slabs, &s_missing, s_count);
  }
}

// Joins the pieces of every query: DP / 4 lanes hold four dims each of a (row,
// head), SUB groups of them every SUB-th piece. The prefix pieces are on their way
// before the row's length is known. A
// query left non-finite, and not by a missing page (whose NaN is the
// denominator's too), is attended once more by its wave on the VALU: on the matrix
// cores a key that a query does not attend has weight 0, and 0 * Inf or 0 * NaN of
// its V is NaN, and so is the 0 * Inf of a weight's low part.
constexpr int kMergeThreads = 256;
// From this many pieces on several groups of lanes share a (row, head): 8 requests behind
// 8192 tokens (32 pieces) 15.8 us with it, 18.7 without; 16 prompts of fp32 (3) 41 without,
// 44 with it. Between 4 and 16 it makes no difference.
constexpr int kManyPieces = 8;

// Pieces joined so far: four dims of the accumulators, maximum, denominator.
struct Joined {
  float m = -INFINITY, l = 0.f;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float2 ml, const float4& v) {
    const float top = fmaxf(m, ml.x);
    const float wo = m == -INFINITY ? 0.f : fast_exp2(m - top);
    const float wn = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
    l = fmaf(l, wo, ml.y * wn);  // a NaN denominator stays
    acc.x = fmaf(acc.x, wo, v.x * wn); acc.y = fmaf(acc.y, wo, v.y * wn);
    acc.z = fmaf(acc.z, wo, v.z * wn); acc.w = fmaf(acc.w, wo, v.w * wn);
    m = top;
  }
};

template <int DT, int DP, int SUB>
__global__ __launch_bounds__(kMergeThreads) void shared_merge_kernel(SharedArgs a, Plan p) {
  using T = typename Elem<DT>::T;
  constexpr int LANES = DP / 4, PER = kMergeThreads / (LANES * SUB);  // pairs a workgroup
  __shared__ int s_count[kMergeThreads / kWave];
  const Geometry& g = a.g;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int64_t pair0 = int64_t(blockIdx.x) * PER, pair = pair0 + tid / (LANES * SUB);
  const int64_t row = pair / g.heads;
  const int head = int(pair - row * g.heads), dd = 4 * (lane % LANES), sub = lane / LANES % SUB;
  const float* base = p.partials + (int64_t(head) * a.rows + row) * part_row<DP>();
  const int64_t step = int64_t(g.heads) * a.rows * part_row<DP>();
  Joined all;
  auto join = [&](int first, int end) {
#pragma unroll 4
    for (int s = first + sub; s < end; s += SUB) {
      const float* x = base + s * step;
      all.add(*reinterpret_cast<const float2*>(x + DP), *reinterpret_cast<const float4*>(x + dd));
    }
  };
  if (row < a.rows) join(0, pieces_of(p, head * p.tiles + int(row) / (32 * p.qt)));
  int r = int(row);
  if (a.cu_tokens) {
    // the request of the workgroup's first row: as many as start at or before it,
    // less one; of a later row by bisection from there
    const int64_t row0 = pair0 / g.heads;
    int n = 0;
    for (int j = tid; j < a.b; j += kMergeThreads) n += a.cu_tokens[j] <= row0;
#pragma unroll
    for (int w = kWave / 2; w > 0; w /= 2) n += __shfl_xor(n, w);
    if (lane == 0) s_count[wave] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kMergeThreads / kWave; ++w) n += s_count[w];
    r = max(n - 1, 0);
    if (row < a.rows && r + 1 < a.b && a.cu_tokens[r + 1] <= row) {
      int above = a.b;
      while (r + 1 < above) {
        const int mid = (r + above) / 2;
        if (a.cu_tokens[mid] <= row) r = mid;
        else above = mid;
      }
    }
  }
  // what the row attends: nothing where it is no request's (`write` false)
  Request rq{0, 0, 0};
  if (row < a.rows) rq = request_of(a, r);
  const int i = int(row - rq.row0);
  const bool write = row < a.rows && row >= rq.row0 && i < rq.tokens;
  const int64_t keys = int64_t(rq.length) + i + 1, cap = int64_t(g.columns) * g.page_size;
  T* const out = static_cast<T*>(a.out) + row * a.o_r + int64_t(head) * g.dim;
  bool redo = false;
  if (write && (rq.length < 0 || keys > cap)) {
    // padding, or a token past the table
    if (sub == 0 && dd < g.dim) {
      const float x = rq.length < 0 ? 0.f : NAN;
      store4<DT>(out + dd, x, x, x, x);
    }
  } else if (write) {
    const int tq = 32 * p.own_qt;
    const int64_t end = a.k ? keys : min(int64_t(rq.length) + min((i / tq + 1) * tq, rq.tokens), cap + 1);
    join(p.pieces, p.pieces + int((end + p.split_keys - 1) / p.split_keys));
#pragma unroll
    for (int w = LANES; w < LANES * SUB; w <<= 1)
      all.add(float2{__shfl_xor(all.m, w), __shfl_xor(all.l, w)},
              float4{__shfl_xor(all.acc.x, w), __shfl_xor(all.acc.y, w), __shfl_xor(all.acc.z, w), __shfl_xor(all.acc.w, w)});
    const float zero = fmaf(all.acc.x, 0.f, all.acc.y * 0.f) + fmaf(all.acc.z, 0.f, all.acc.w * 0.f);
    redo = isnan(zero) && !isnan(all.l);
    if (sub == 0 && dd < g.dim) {
      const float inv = inverse(all.l);
      store4<DT>(out + dd, divided<DT>(all.acc.x, all.l, inv), divided<DT>(all.acc.y, all.l, inv),
                 divided<DT>(all.acc.z, all.l, inv), divided<DT>(all.acc.w, all.l, inv));
    }
  }
  uint64_t left = __ballot(redo);
  if (left) __threadfence_block();  // the stores above come before those that repeat them
  while (left) {
    const int first = __builtin_ctzll(left) / (LANES * SUB) * (LANES * SUB);
    left &= LANES * SUB == kWave ? 0 : ~(((uint64_t(1) << (LANES * SUB & 63)) - 1) << first);
    const int64_t again = __shfl(row, first), n = __shfl(keys, first);
    const int h = __shfl(head, first), req = __shfl(r, first);
    const T* q = static_cast<const T*>(a.q) + again * a.q_r + int64_t(h) * g.dim;
    const T* fk = a.k ? static_cast<const T*>(a.k) + again * a.q_r + int64_t(h) * g.dim : nullptr;
    const T* fv = a.k ? static_cast<const T*>(a.v) + again * a.q_r + int64_t(h) * g.dim : nullptr;
    Walk<DT> w;
    w.keys(q, a.slabs, a.prefix_table, a.prefix_columns, 0, a.prefix, nullptr, nullptr, g, h, a.qscale);
    w.keys(q, a.slabs, a.table + int64_t(req) * g.columns, g.columns, 0, n, fk, fv, g, h, a.qscale);
    const float l = w.denominator();
    T* const to = static_cast<T*>(a.out) + again * a.o_r + int64_t(h) * g.dim;
    if (lane < g.dim) to[lane] = from_f32<DT>(finalize(w.acc[0], l));
    if (lane + kWave < g.dim) to[lane + kWave] = from_f32<DT>(finalize(w.acc[1], l));
  }
}

// ------------------------------------------------------------------- host ---
bool shared_shape(int b, int rows, int max_tokens, int h, int d, int page_size, int pps, int num_slabs, int prefix,
                  int columns, int layer, int layers, int dtype) {
  return b > 0 && b <= 65535 && rows > 0 && max_tokens > 0 && max_tokens <= rows && h > 0 && d > 0 && d <= 128 &&
         int64_t(b) * h <= 65535 && int64_t(rows) * h * d <= INT32_MAX && (page_size == 8 || page_size == 16 || page_size == 32) &&
         pps > 0 && num_slabs > 0 && int64_t(pps) * num_slabs <= INT32_MAX && prefix >= 0 && columns > 0 &&
         int64_t(b) * columns <= INT32_MAX && int64_t(columns) * page_size <= INT32_MAX - 4096 &&
         int64_t(prefix) <= INT32_MAX - 32768 - int64_t(columns) * page_size && layers > 0 && layer >= 0 && layer < layers &&
         dtype >= 0 && dtype <= 2;
}

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }

// How a launch is cut.
Plan make_plan(int rows, int b, int h, int d, int page_size, int prefix, int columns, int max_tokens, int dtype, bool decode) {
  const int cus = device_compute_units() > 0 ? device_compute_units() : 256;
  const int row_bytes = (d <= 64 ? 64 : 128) * (dtype == kF32 ? 4 : 2);
  const bool wide = !decode && dtype != kF32 && rows > 128;
  const int waves = shape_waves(row_bytes, wide);
  const int slots = (row_bytes * waves <= 1024 ? 2 : 1) * cus;  // workgroups that are resident at once
  const int64_t cap = int64_t(columns) * page_size, bh = int64_t(b) * h;
  Plan p{};
  p.waves = waves;
  // Prefix tiles: the queries' groups of 32 over tiles of 1, 2, 4 or 8 groups,
  // where a tile costs its groups and about one more (us in tiles of 1, 2, 4, 8: 64
  // requests behind 2048 tokens 20.6, 16.7, 17.7, 17.9; 160 rows behind 2048 23.1,
  // 22.0, 20.7, 19.6). Beside streams of own keys two tiles of 4 do as well as a full one of
  // 8 or better (256 requests behind 16001 tokens 68 and 74, 400 behind 1000 154 and 160,
  // 512 of contexts up to 8192 behind 8192 323 and 319), but not those of 240 (47 and 45)
  // nor prompts' (8 of 300-500 behind 8000 213 and 179).
  // fp32 products are slow, so that waves without queries cost more there: groups count three
  // times (with that and without, 6 prompts of 9-37 x 25 behind 3546 54 and 65, 75 requests x
  // 25 of 32 behind 12684 83 and 90, 66 x 12 behind 4000 36 and 33).
  int64_t best = INT64_MAX;
  const int most = decode && row_bytes == 128 && rows >= 256 ? 4 : waves;
  for (int qt = 1; qt <= most; qt *= 2) {
    const int64_t cost = ceil_div(rows, 32 * qt) * ((dtype == kF32 ? 3 * qt : qt) + 1);
    if (cost <= best) { best = cost; p.qt = qt; }
  }
  // Smaller ones where the prefix is too short for an item on each compute unit (decode 257 x
  // 12 behind 199 tokens 14.6 us, 18.6 without; prompts gain and lose by it).
  while (decode && p.qt > 1 && ceil_div(rows, 32 * p.qt) * h * ceil_div(prefix, 64) < cus) p.qt /= 2;
  p.tiles = int(ceil_div(rows, 32 * p.qt));
  if (prefix > 0) {
    // Units of a staged half. One item a compute unit, which leaves half of its
    // places (a quarter of the compute units, where an item takes a whole one) to
    // the own items; tiles of few queries wait for memory more than they compute
    // and fill every place. us, items of half as many, as many and twice as many
    // compute units: 256 decode rows x 16 heads behind 16001 tokens 88, 76 and 94; 64
    // requests of 1-20 tokens x 12 behind 4096 50, 42 and 49; one decode row x 12
    // behind 32000 40, 29 and 27; 24 prompts x 16 heads of 128 behind 8100 (eight waves)
    // 358, 378 and 390, with three quarters 356.
    // Where the own items are few (they fit beside each other), prefix items take every
    // place too: 16 prompts of 256-512 behind 2048 105 us instead of 120.
    // Pieces of 256 keys at least unless few would be left (4 rows fp32 x 12 heads behind
    // 200: 10.5 in pieces of 64, 13 whole), cut at the tiles' ends where that keeps nine
    // tenths of the items busy, for the fewest pieces.
    const int64_t head_tiles = int64_t(p.tiles) * h;
    const int64_t own = decode ? INT64_MAX : bh * ceil_div(max_tokens, 256) * ceil_div(cap + 1, 2048);
    const int64_t want = 2 * p.qt < waves || (row_bytes == 128 && own <= slots) ? slots
                         : slots > cus || dtype == kF32                         ? cus
                                                                                : 3 * int64_t(cus) / 4;
    p.prefix_unit = row_bytes == 128 ? 128 : 64;
    int64_t units = ceil_div(prefix, p.prefix_unit);
    if (head_tiles * ceil_div(prefix, 256) < cus / 4) {
      p.prefix_unit = 64;
      units = ceil_div(prefix, 64);
      p.item_units = 1;
    } else {
      p.item_units = int(std::max<int64_t>(256 / p.prefix_unit, ceil_div(head_tiles * units, want)));
    }
    p.item_units = int(std::min<int64_t>(p.item_units, int64_t(kPages) * page_size / p.prefix_unit));
    const int64_t even = ceil_div(units, ceil_div(units, p.item_units));  // units of pieces of one length
    const int64_t items = head_tiles * ceil_div(units, even), rounds = ceil_div(items, want);
    if (10 * items >= 9 * rounds * want || even == units) {
      p.item_units = int(even);
      units = ceil_div(units, even) * even;
    }
    p.tile_units = int(units);
    p.units = head_tiles * units;
    p.prefix_items = ceil_div(p.units, p.item_units);
    p.pieces = int(units % p.item_units == 0   ? units / p.item_units
                   : p.item_units % units == 0 ? 1
                                               : (units - 2) / p.item_units + 2);
  }
  if (decode) {
    // More waves for a (request, head) where there are few of them: us with 2, 4 and 8
    // waves, 64 x 12 17.2, 16.8, 20.4; 128 x 16 48, 45, 56; 256 x 16 77.6, 83, 97;
    // 512 x 25 322, 340, 431.
    const int64_t resident = int64_t(slots) * waves;
    p.item_waves = bh * 8 <= resident ? 8 : bh * 4 <= 2 * resident ? 4 : 2;
    p.item_waves = std::min(p.item_waves, waves);
    // A wave has eight tokens at least, where there are many rows 64 (512 x 12 behind 4096 and
    // own contexts up to 64: 38 us with one wave, 41 with two).
    const int least = bh > resident ? 64 : 8;
    while (p.item_waves > 1 && (p.item_waves - 1) * least >= cap) p.item_waves /= 2;
    // Splits of 512 tokens: a wave resolves the page of each of its steps into one
    // lane, 64 steps of 8 tokens. Longer ones for tables of more than 64.
    p.split_keys = int(std::min<int64_t>(512 * p.item_waves, std::max<int64_t>(512, ceil_div(cap, 64 * 64) * 64)));
    p.splits = int(ceil_div(cap, p.split_keys));
    const int groups = waves / p.item_waves;
    p.more_blocks = p.splits > 1 ? int(std::min<int64_t>(slots, ceil_div(bh * p.splits, groups))) : 0;
    p.own_blocks = ceil_div(bh, groups);
    p.own_qt = 1;
  } else {
    p.own_qt = std::min(waves, max_tokens <= 32 ? 1 : max_tokens <= 64 ? 2 : max_tokens <= 128 ? 4 : 8);
    p.own_tiles = int(ceil_div(max_tokens, 32 * p.own_qt));
    p.split_keys = 2048;
    p.splits = int(ceil_div(cap + 1, p.split_keys));
    p.own_blocks = bh * p.own_tiles * p.splits;
    // (256 requests of 1-8 tokens, 15400 bounds: 213 us listed, 240 not; 64 of 5, 3840: 33 and 32)
    p.listed = p.own_blocks > 8 * slots;
    if (p.listed) p.own_blocks = 8 * slots;
  }
  return p;
}

// Whether the launches can hold the plan's workgroups (2^32 threads), and the counts of
// items their 32 bits.
bool plan_fits(const Plan& p, int rows, int h) {
  return p.units < (int64_t(1) << 31) - p.item_units && p.prefix_items < 1 << 22 && int64_t(rows) * h < 1 << 26 &&
         int64_t(p.own_tiles) * p.splits < 1 << 22;
}

size_t plan_bytes(const Plan& p, int rows, int h, int d) {
  return size_t(p.pieces + p.splits) * h * rows * (d <= 64 ? part_row<64>() : part_row<128>()) * sizeof(float);
}

// Rows that the fast path takes: whole 16-byte chunks.
bool whole_chunks(int d, int dtype) { return d * (dtype == kF32 ? 4 : 2) % 16 == 0; }

template <int DT, int DP, int W, Rows FULL>
void launch_tiles(const SharedArgs& a, const Plan& p) {
  const int blocks = int(p.prefix_items + p.own_blocks);
  if (p.listed) shared_kernel<DT, DP, W, FULL, kOwnListed><<<blocks, W * kWave>>>(a, p);
  else shared_kernel<DT, DP, W, FULL, kOwnTiles><<<blocks, W * kWave>>>(a, p);
}

template <int DT, int DP, Rows FULL>
void launch_rows(const SharedArgs& a, const Plan& p) {
  constexpr int W = shape_waves(DP * elem_bytes<DT>(), false);
  if (a.k) shared_kernel<DT, DP, W, FULL, kOwnToken><<<int(p.prefix_items + p.more_blocks + p.own_blocks), W * kWave>>>(a, p);
  else if (p.waves == W) launch_tiles<DT, DP, W, FULL>(a, p);
  else if constexpr (W == 4 && DT != kF32) launch_tiles<DT, DP, 8, FULL>(a, p);
}

template <int DT, int DP>
void launch_fast(const SharedArgs& a, const Plan& p) {
  if (a.g.dim == DP) launch_rows<DT, DP, kRowsFull>(a, p);
  else launch_rows<DT, DP, kRowsPadded>(a, p);
  const int64_t pairs = int64_t(a.rows) * a.g.heads;
  constexpr int LANES = DP / 4;
  if (p.pieces >= kManyPieces) shared_merge_kernel<DT, DP, kWave / LANES><<<int(ceil_div(pairs, kMergeThreads / kWave)), kMergeThreads>>>(a, p);
  else shared_merge_kernel<DT, DP, 1><<<int(ceil_div(pairs, kMergeThreads / LANES)), kMergeThreads>>>(a, p);
}

hipError_t launch_shared(SharedArgs& a, int dtype, void* workspace) {
  const int es = dtype == kF32 ? 4 : 2;
  auto rows16 = [&](int64_t x) { return x * es % 16 == 0; };
  if (whole_chunks(a.g.dim, dtype) && rows16(a.q_r) && rows16(a.o_r) && aligned16(a.out) && aligned16(a.q) &&
      (!a.k || (aligned16(a.k) && aligned16(a.v)))) {
    Plan p = make_plan(a.rows, a.b, a.g.heads, a.g.dim, a.g.page_size, a.prefix, a.g.columns, a.max_tokens, dtype, a.k != nullptr);
    p.partials = static_cast<float*>(workspace);
#define MT_FAST(DT)                       \
  if (a.g.dim <= 64) launch_fast<DT, 64>(a, p); \
  else launch_fast<DT, 128>(a, p);
    if (dtype == kF32) { MT_FAST(kF32) }
    else if (dtype == kF16) { MT_FAST(kF16) }
    else { MT_FAST(kBF16) }
#undef MT_FAST
    return hipGetLastError();
  }
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
  size_t need = 0;
  for (int decode = 0; whole_chunks(d, dtype) && decode < (max_tokens == 1 && rows == b ? 2 : 1); ++decode) {
    const Plan p = make_plan(rows, b, h, d, page_size, prefix_tokens, columns, max_tokens, dtype, decode);
    if (!plan_fits(p, rows, h)) return hipErrorInvalidValue;
    need = std::max(need, plan_bytes(p, rows, h, d));
  }
  *bytes = need;
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
  return launch_shared(a, dtype, workspace);
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
  return launch_shared(a, dtype, workspace);
}

}  // extern "C"
