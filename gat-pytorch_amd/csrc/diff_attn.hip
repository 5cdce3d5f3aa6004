// Differential attention over the in-neighbours of every node, and the learned relative position
// bias its logits can carry:
//   x_m[e,h] = scale q[i,h,m] . k[j,h,m] + bias[bucket[e],h]        (e = j -> i, m = 1, 2)
//   out[i,h] = sum_e (p_1 - lam_h p_2) v[j,h],   p_m = softmax of x_m over i's edges
// Backward, with w = p_1 - lam p_2, dw_e = go[i] . v[j], D_m = sum_e p_m dw:
//   dx_1 = p_1 (dw - D_1),  dx_2 = -lam p_2 (dw - D_2)
//   gq_m[i] = scale sum_e dx_m k_m[j];  gk_m[j] = scale sum_e dx_m q_m[i];  gv[j] = sum_e w go[i]
//   glam_h = -sum_i D_2;  gbias[b,h] = sum over b's edges of dx_1 + dx_2
//
// Bound by the gathers: every edge reads (2d + dv) elements of its source's (or destination's) row
// per head, from L2 as long as one head's rows of the nodes in flight fit there. So a work item is
// (row, head), items run in chunks of kChunk rows one head after the other, and whole (chunk, head)
// units go to one XCD. The products are sparse (a row's neighbours are shared with no other row),
// so they run on the vector units, packed dot products for bf16, every sum in fp32.
//
// G lanes hold one edge's row: lane c of them the c-th 8-element chunk (of both maps; chunks c and c
// + G of the values). What an edge needs once (its index, logits, weights) is held by one lane
// each, NL = min(G, 16) edges at a time, and handed to the G lanes by a broadcast within their 16
// lanes; a tile's dot products are summed over the lanes by a reduce-scatter that leaves edge i's
// with lane i. So every step but the multiply-adds over a row costs 1 / NL of an instruction per
// edge and lane. 64 / G edges are in flight per wave; a row has gs = 16, 32 or 64 lanes (gs / G slots
// of edges side by side, joined at its end).
// Forward: the logits and each row's statistics (gathers k), then the weighted values (gathers v).
// Backward: A: dw and D (v); B: gq, and {scale dx_1, scale dx_2, w} of each edge (k); C: gk and gv by
// the transposed CSR (q and go). One gather a pass keeps a head's gathered rows of a graph inside
// L2, and the sums of pieces (rows of more than hub_edges edges) are plain. A serving call takes
// one kernel with a running softmax instead: its rows are cut into pieces whose partial results
// carry their maxima, and it needs no array of logits. Every sum has a fixed order.
//
// 44 900 nodes, 1.27 M edges, 4 heads, bf16 d = 128, dv = 256: logits 198 us, values 168, A 160, B
// 190, C 370 (2.6 GB gathered by each, 5.2 GB by C: 13 to 16 TB/s, 74 to 87% of it from L2). The
// vector units issue 0.85 instructions a cycle and CU in the values pass, 0.7 in B and C, 0.55 in
// the dot products.
// One node of 65 537 edges, 8 heads, bf16 d = 64, dv = 128: 48 us and 7 for the join = 5.5 TB/s.
#include "dtypes.h"

namespace gatx {
namespace {

constexpr int kChunk = 2048;       // rows of a (chunk, head) unit
constexpr int kWantWaves = 4096;   // 4 a SIMD
constexpr int kMaxD = 256, kMaxDv = 512, kMaxBuckets = 256;
constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.44269504088896341f;

// ------------------------------------------------------------------ 8 elements of a row
template <typename T>
struct Raw {
  uint4 v;
};
template <>
struct Raw<float> {
  float4 a, b;
};
template <typename T>
__device__ inline Raw<T> load8(const T* p) {
  Raw<T> r;
  r.v = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <>
__device__ inline Raw<float> load8<float>(const float* p) {
  Raw<float> r;
  r.a = *reinterpret_cast<const float4*>(p);
  r.b = *reinterpret_cast<const float4*>(p + 4);
  return r;
}
// From any address (global loads need no alignment).
template <typename T>
__device__ inline Raw<T> load8_anywhere(const T* p) {
  Raw<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T>
__device__ inline Raw<T> keep8(bool keep, Raw<T> x) {
  x.v.x = keep ? x.v.x : 0u;
  x.v.y = keep ? x.v.y : 0u;
  x.v.z = keep ? x.v.z : 0u;
  x.v.w = keep ? x.v.w : 0u;
  return x;
}
__device__ inline Raw<float> keep8(bool keep, Raw<float> x) {
  x.a = make_float4(keep ? x.a.x : 0.f, keep ? x.a.y : 0.f, keep ? x.a.z : 0.f, keep ? x.a.w : 0.f);
  x.b = make_float4(keep ? x.b.x : 0.f, keep ? x.b.y : 0.f, keep ? x.b.z : 0.f, keep ? x.b.w : 0.f);
  return x;
}

// Elements [from, 8) alone.
template <typename T>
struct From {
  uint32_t m[2 * sizeof(T)];
  __device__ From(int from) {
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) {
      if (sizeof(T) == 4) m[i] = i >= from ? ~0u : 0u;
      else m[i] = (2 * i >= from ? 0xffffu : 0u) | (2 * i + 1 >= from ? 0xffff0000u : 0u);
    }
  }
  __device__ Raw<T> operator()(const Raw<T>& x) const {
    uint32_t w[2 * sizeof(T)];
    __builtin_memcpy(w, &x, sizeof(w));
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) w[i] &= m[i];
    Raw<T> r;
    __builtin_memcpy(&r, w, sizeof(r));
    return r;
  }
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
__device__ inline float dot2(__bf16, uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a),
                                         __builtin_bit_cast(bf16x2, b), c, false);
}
// fp16: two mixed-precision multiply-adds, each rounded once. The packed fp16 dot product is less
// exact: a sum of D_2 over 44 900 rows came out 1e-6 to 1e-5 off, against 1e-7 this way (and with
// bf16's packed product).
__device__ inline float dot2(_Float16, uint32_t a, uint32_t b, float c) {
  const f16x2 x = __builtin_bit_cast(f16x2, a), y = __builtin_bit_cast(f16x2, b);
  return fmaf((float)x.y, (float)y.y, fmaf((float)x.x, (float)y.x, c));
}
template <typename T>
__device__ inline float dot8(const Raw<T>& a, const Raw<T>& b, float c) {
  c = dot2(T(), a.v.x, b.v.x, c);
  c = dot2(T(), a.v.y, b.v.y, c);
  c = dot2(T(), a.v.z, b.v.z, c);
  return dot2(T(), a.v.w, b.v.w, c);
}
__device__ inline float dot8(const Raw<float>& a, const Raw<float>& b, float c) {
  c = fmaf(a.a.x, b.a.x, c);
  c = fmaf(a.a.y, b.a.y, c);
  c = fmaf(a.a.z, b.a.z, c);
  c = fmaf(a.a.w, b.a.w, c);
  c = fmaf(a.b.x, b.b.x, c);
  c = fmaf(a.b.y, b.b.y, c);
  c = fmaf(a.b.z, b.b.z, c);
  return fmaf(a.b.w, b.b.w, c);
}

__device__ inline float2 unpack2(__bf16, uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ inline float2 unpack2(_Float16, uint32_t x) {
  const f16x2 h = __builtin_bit_cast(f16x2, x);
  return make_float2((float)h.x, (float)h.y);
}
template <typename T>
__device__ inline void unpack8(const Raw<T>& x, float (&f)[8]) {
  const uint32_t w[4] = {x.v.x, x.v.y, x.v.z, x.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = unpack2(T(), w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ inline void unpack8(const Raw<float>& x, float (&f)[8]) {
  f[0] = x.a.x; f[1] = x.a.y; f[2] = x.a.z; f[3] = x.a.w;
  f[4] = x.b.x; f[5] = x.b.y; f[6] = x.b.z; f[7] = x.b.w;
}
// Whether an edge's row counts, as unpacking uses it: bf16 pairs are unpacked by one instruction an
// element that can also clear it (the mask of the upper half, the byte selector of the lower).
template <typename T>
struct Keep {
  int keep;
  __device__ Keep(bool open) : keep(open) {}
  template <int G, int I>
  __device__ Keep of_edge() const;
  __device__ void unpack(const Raw<T>& x, float (&f)[8]) const { unpack8(keep8(keep != 0, x), f); }
};
template <>
struct Keep<__bf16> {
  int hi, sel;
  __device__ Keep(bool open) : hi(open ? (int)0xffff0000u : 0), sel(open ? 0x01000c0c : 0x0c0c0c0c) {}
  template <int G, int I>
  __device__ Keep of_edge() const;
  __device__ void unpack(const Raw<__bf16>& x, float (&f)[8]) const {
    const uint32_t w[4] = {x.v.x, x.v.y, x.v.z, x.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(__builtin_amdgcn_perm(w[i], w[i], (uint32_t)sel));
      f[2 * i + 1] = __uint_as_float(w[i] & (uint32_t)hi);
    }
  }
};
__device__ inline void axpy8(float p, const float (&x)[8], float (&acc)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = fmaf(p, x[i], acc[i]);
}
template <typename T>
__device__ inline void axpy8(float p, const Raw<T>& x, float (&acc)[8]) {
  float f[8];
  unpack8(x, f);
  axpy8(p, f, acc);
}
// Columns [at, at + 8) of a packed row of `width` elements; !whole: rows that are aligned to an
// element only and can end inside the 8.
template <typename T>
__device__ inline void store8(T* row, int at, int width, bool whole, const float (&x)[8]) {
  if (whole) {
    if (at >= width) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + at) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(row + at + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      store_f32<T, 8>(row + at, x);
    }
  } else if (at + 8 <= width) {
    T y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (T)x[i];
    __builtin_memcpy(row + at, y, sizeof(y));   // global stores need no alignment
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < width) row[at + i] = (T)x[i];
  }
}

// ------------------------------------------------------------------ lanes of a wave
// Sums over the G lanes of an edge.
template <int G>
__device__ inline float edge_sum(float v) {
  return group_sum<G>(v);
}
// Sums over the slots of a row (lanes l, l + G, ... of its gs >= 16), in every lane: rotations inside
// 16 lanes, swaps beyond.
template <int G, int N>
__device__ inline void slots_sum(float (&v)[N], int gs) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (G <= 8) v[i] += dpp<0x128>(v[i]);   // row_ror:8
    if (G <= 4) v[i] += dpp<0x124>(v[i]);
    if (G <= 2) v[i] += dpp<0x122>(v[i]);
    if (G <= 1) v[i] += dpp<0x121>(v[i]);
  }
  if (G <= 16 && gs >= 32) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false,
                                                false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  }
  if (gs >= 64) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false,
                                                false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  }
}
template <int G>
__device__ inline float slots_max(float v, int gs) {
  for (int d = G; d < gs; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
__device__ inline int wave_max(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, __shfl_xor(v, d));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ inline float exp_(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// Edges per tile and slot: one for each lane of an edge, 16 at most (what a DPP row spans).
template <int G>
constexpr int kTile = G < 16 ? G : 16;
// x of the lane that holds edge I of the own slot's tile.
template <int G, int I>
__device__ inline int tile_get(int x) {
  if constexpr (G >= 16) {
    return __builtin_amdgcn_update_dpp(x, x, 0x150 + I, 0xf, 0xf, false);   // row_newbcast:I
  } else if constexpr (G == 8) {
    const int lo = __builtin_amdgcn_update_dpp(x, x, 0x150 + I, 0xf, 0x3, false);
    return __builtin_amdgcn_update_dpp(lo, x, 0x158 + I, 0xf, 0xc, false);
  } else if constexpr (G == 4) {
    return __builtin_amdgcn_update_dpp(x, x, I * 0x55, 0xf, 0xf, false);   // quad_perm:[I,I,I,I]
  } else if constexpr (G == 2) {
    return __builtin_amdgcn_update_dpp(x, x, I ? 0xF5 : 0xA0, 0xf, 0xf, false);
  } else {
    return x;
  }
}
template <int G, int I>
__device__ inline float tile_get(float x) {
  return __int_as_float(tile_get<G, I>(__float_as_int(x)));
}
template <int G, int I>
__device__ inline int64_t tile_get(int64_t x) {
  const uint32_t lo = (uint32_t)tile_get<G, I>((int)x);
  return ((int64_t)tile_get<G, I>((int)(x >> 32)) << 32) | lo;
}
template <typename T>
template <int G, int I>
__device__ inline Keep<T> Keep<T>::of_edge() const {
  Keep k = *this;
  k.keep = tile_get<G, I>(keep);
  return k;
}
template <int G, int I>
__device__ inline Keep<__bf16> Keep<__bf16>::of_edge() const {
  Keep k = *this;
  k.hi = tile_get<G, I>(hi);
  k.sel = tile_get<G, I>(sel);
  return k;
}
template <bool ALL, typename T>
__device__ inline void axpy_kept(float p, const Raw<T>& x, const Keep<T>& k, float (&acc)[8]) {
  float f[8];
  if (ALL) unpack8(x, f);
  else k.unpack(x, f);
  axpy8(p, f, acc);
}
// A gathered row's offset and where it is: in bytes for the 16-bit types (an instruction less a load),
// in elements for float32 (PPI, d = 61: logits 353 us, 365 in bytes).
template <typename T>
__device__ inline int64_t row_off(int64_t j, int64_t ld) {
  return j * ld * (sizeof(T) == 2 ? 2 : 1);
}
template <typename T>
__device__ inline const T* row_at(const T* p, int64_t off) {
  return sizeof(T) == 2 ? (const T*)((const char*)p + off) : p + off;
}
// Sums of a tile's values over the G lanes of an edge: the lane that holds edge i gets v[i]'s.
template <int G>
__device__ inline float tile_scatter(float (&v)[kTile<G>], int lane) {
  constexpr int N = kTile<G>;
  auto level = [&](auto B, auto ctrl) {   // partners differ in lane bit B (and agree on the halves)
    constexpr int half = 1 << decltype(B)::value;
    if constexpr (half < N) {
      const bool up = lane & half;
#pragma unroll
      for (int j = 0; j < half; ++j) {
        const float send = up ? v[j] : v[half + j], keep = up ? v[half + j] : v[j];
        v[j] = keep + dpp<decltype(ctrl)::value>(send);
      }
    }
  };
  level(std::integral_constant<int, 3>(), std::integral_constant<int, 0x140>());
  level(std::integral_constant<int, 2>(), std::integral_constant<int, 0x141>());
  level(std::integral_constant<int, 1>(), std::integral_constant<int, 0x4E>());
  level(std::integral_constant<int, 0>(), std::integral_constant<int, 0xB1>());
  if constexpr (G == 32) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[0]), false,
                                              false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v[0];
}
// f(integral_constant 0), ..., f(N - 1)
template <typename F, int... I>
__device__ inline void each_(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ inline void each(F&& f) {
  each_(f, std::make_integer_sequence<int, N>());
}

// ------------------------------------------------------------------ work items
// Which (row, head, edges) a group of `gs` lanes has. Counts are below 2^31 (checked at launch).
struct Work {
  // plain rows: units of 2^chunk_log blocks' rows of one head, dealt to the XCDs in turn
  int rows, heads, gs, gs_log, unit_log;
  int units;                       // row chunks * heads
  const int32_t* rowptr;
  const int4* order;               // rows of like length side by side (row_order_kernel), or NULL
  // pieces: of hub rows (hubs != NULL: the plan's entries), or of the rows of a serving call
  // (nodes != NULL: `pieces` of each)
  int hub_edges;
  const int32_t *hubs, *hub_count;
  int hub_bound, hub_blocks;       // blocks [0, hub_blocks) have the pieces
  const int64_t* nodes;
  int pieces;
  int64_t num_nodes;
};
struct Item {
  int row;        // of the outputs and of q; < 0: none
  int slot;       // of the partial results; < 0: this item is the whole row
  int head, beg, n;   // its edges: n from beg on
  bool bad;       // a node id that does not exist
};
__device__ inline Item find_item(const Work& w) {
  const int grp_log = 8 - w.gs_log, grp = (int)threadIdx.x >> w.gs_log;
  Item it = {-1, -1, 0, 0, 0, false};
  if (w.nodes) {
    const uint32_t i = (blockIdx.x << grp_log) + grp, rh = i / (uint32_t)w.pieces;
    const uint32_t row = rh / (uint32_t)w.heads;
    if (row >= (uint32_t)w.rows) return it;
    it.row = (int)row;
    it.head = (int)(rh - row * w.heads);
    const int piece = (int)(i - rh * w.pieces);
    it.slot = w.pieces > 1 ? it.row * w.pieces + piece : -1;
    const int64_t n = w.nodes[it.row];
    it.bad = n < 0 || n >= w.num_nodes;
    if (it.bad) return it;
    const int b = w.rowptr[n], deg = w.rowptr[n + 1] - b;
    const int64_t len = ((int64_t)deg + w.pieces - 1) / w.pieces, at = min((int64_t)deg, piece * len);
    it.beg = b + (int)at;
    it.n = (int)min(len, deg - at);
    return it;
  }
  if ((int)blockIdx.x < w.hub_blocks) {
    const uint32_t i = (blockIdx.x << grp_log) + grp, pc = i / (uint32_t)w.heads;
    if (pc >= (uint32_t)w.hub_bound || (int)pc >= *w.hub_count) return it;
    const int32_t* hp = w.hubs + 4 * (int64_t)pc;
    it.row = hp[0];
    it.head = (int)(i - pc * w.heads);
    it.slot = (int)pc;
    const int b = w.rowptr[it.row], deg = w.rowptr[it.row + 1] - b, at = hp[1] * w.hub_edges;
    it.beg = b + at;
    it.n = min(w.hub_edges, deg - at);
    return it;
  }
  const uint32_t b = blockIdx.x - w.hub_blocks, j = b >> 3;
  const uint32_t unit = (j >> w.unit_log << 3) + (b & 7);
  if (unit >= (uint32_t)w.units) return it;
  const uint32_t ck = unit / (uint32_t)w.heads;
  const uint32_t block = (ck << w.unit_log) + (j & ((1u << w.unit_log) - 1));
  const uint32_t row = (block << grp_log) + grp;
  if (row >= (uint32_t)w.rows) return it;
  it.head = (int)(unit - ck * w.heads);
  int node = (int)row, n;
  if (w.order) {
    const int4 o = w.order[row];
    node = o.x;
    it.beg = o.y;
    n = o.z;
  } else {
    it.beg = w.rowptr[row];
    n = w.rowptr[row + 1] - it.beg;
  }
  if (w.hub_edges > 0 && n > w.hub_edges) return it;   // in pieces, above
  it.n = n;
  it.row = node;
  return it;
}

// The rows of each chunk by falling length: {row, first edge, edges, -}. The rows that share a wave
// step through their edges together, so a wave takes as long as its longest. A stable counting sort
// of 2048 rows by pairs of edges, a workgroup each: equal rows keep their order (and what they share
// of the first-level caches). No result depends on it: a row's own lanes and their order stay. (PPI
// batch, bf16 d = 128, dv = 256: logits 205 -> 197 us, values 186 -> 168, dw 166 -> 159, gq 213 -> 201,
// gk and gv 397 -> 371.)
constexpr int kOrderKeys = 512, kOrderWaves = 16, kOrderBatches = kChunk / (64 * kOrderWaves);
__global__ void __launch_bounds__(64 * kOrderWaves) row_order_kernel(const int32_t* rowptr,
                                                                     int64_t rows, int4* order) {
  // how many rows of a key a wave has, then where its first one goes
  __shared__ int at[kOrderKeys][kOrderWaves];
  __shared__ int sums[kOrderWaves];
  constexpr int N = kOrderKeys * kOrderWaves, own = N / (64 * kOrderWaves);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < N; i += 64 * kOrderWaves) (&at[0][0])[i] = 0;
  const int64_t r0 = (int64_t)blockIdx.x * kChunk, first = r0 + wave * (64 * kOrderBatches) + lane;
  int beg[kOrderBatches], n[kOrderBatches], off[kOrderBatches];
#pragma unroll
  for (int b = 0; b < kOrderBatches; ++b) {
    const int64_t r = min(first + 64 * b, rows - 1);
    beg[b] = rowptr[r];
    n[b] = rowptr[r + 1] - beg[b];
  }
  auto key_of = [](int x) { return kOrderKeys - 1 - min((x + 1) >> 1, kOrderKeys - 1); };
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kOrderBatches; ++b) {
    const bool in = first + 64 * b < rows;
    const int key = key_of(n[b]);
    uint64_t same = __ballot(in);   // the batch's rows of this key
#pragma unroll
    for (int bit = 0; bit < 9; ++bit) {
      const uint64_t m = __ballot((key >> bit) & 1);
      same &= (key >> bit) & 1 ? m : ~m;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), had = at[key][wave];
    off[b] = had + rank;
    wave_lds_sync();
    if (in && rank == 0) at[key][wave] = had + __popcll(same);
    wave_lds_sync();
  }
  __syncthreads();
  // exclusive sums, the keys in order and of each key the waves
  int* mine = &at[0][0] + tid * own;
  int before[own], sum = 0;
#pragma unroll
  for (int i = 0; i < own; ++i) {
    before[i] = sum;
    sum += mine[i];
  }
  int upto = sum;
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int base = upto - sum;
  for (int w = 0; w < wave; ++w) base += sums[w];
#pragma unroll
  for (int i = 0; i < own; ++i) mine[i] = base + before[i];
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kOrderBatches; ++b) {
    const int64_t r = first + 64 * b;
    if (r < rows) order[r0 + at[key_of(n[b])][wave] + off[b]] = make_int4((int)r, beg[b], n[b], 0);
  }
}

struct AttnArgs {
  Work w;
  const void *q, *k, *v, *go;
  int64_t ldq, ldk, ldv, ldgo;
  int64_t q_end;             // elements of an unpacked q; 0: packed
  int kv_plain;              // serving: k and v as they come too
  int d, dv, dp, dvp;
  const int32_t* col;        // (C: scol)
  const int32_t* seid;       // C
  int64_t E;
  float scale;
  const float *lam, *bias;
  const uint8_t* bucket;
  float2* S;                 // [H][E] logits
  float4* stat;              // [H][rows] {max1, 1/sum1, max2, 1/sum2}
  void* out;
  float* part;               // [slot][H][...], [part_width] of the sums
  int part_width;
  // backward
  float* dw;                 // [H][E]
  float2* D;                 // [H][rows]
  float4* rec;               // [H][E] {scale dx1, scale dx2, w, dx1 + dx2}
  void *gq, *gk, *gv;
};

// A lane's place in its row's group, and its chunks' columns. Lanes past a row's last chunk read that
// one again (no branch around a load); their part of a dot product is dropped (in_d, in_dv), and
// what they add up is not stored.
template <int G, int NV>
struct Lane {
  int c, slot, slots, at_d, at_dv[NV];
  bool in_d, in_dv[NV];
  __device__ Lane(int gs, int dp, int dvp) {
    const int lane = threadIdx.x & (gs - 1);
    c = lane & (G - 1);
    slot = lane / G;
    slots = gs / G;
    in_d = c * 8 < dp;
    at_d = min(c * 8, dp - 8);
    for (int i = 0; i < NV; ++i) {
      in_dv[i] = (c + i * G) * 8 < dvp;
      at_dv[i] = min((c + i * G) * 8, dvp - 8);
    }
  }
};
// Chunk `at` of map m of a row of q. Unpacked rows (d as it is, any alignment) are read once a row
// anyway, as whole unaligned chunks whose elements past d are dropped; a chunk that would pass the
// end of q, element by element. (44 900 x 6 heads of d = 61 in float32: packing 160 -> 100 us, the
// logits 335 -> 353.)
template <typename T>
__device__ inline Raw<T> load_q(const AttnArgs& a, int64_t row, int head, int m, int at) {
  if (a.q_end == 0)
    return load8((const T*)a.q + row * a.ldq + (int64_t)(2 * head + m) * a.dp + at);
  const int64_t o = row * a.ldq + (int64_t)(2 * head + m) * a.d + at;
  const T* p = (const T*)a.q + o;
  T x[8];
  if (o + 8 <= a.q_end) {
    __builtin_memcpy(x, p, sizeof(x));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = at + i < a.d ? x[i] : (T)0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = at + i < a.d ? p[i] : (T)0.f;
  }
  Raw<T> r;
  __builtin_memcpy(&r, x, sizeof(r));
  return r;
}
// Turns of `step` edges that cover the longest of the wave's rows.
__device__ inline int turns_of(int n, int step) { return (n + step - 1) / step; }
// Edge number o of an item. Past its end: its first edge again (index 0 of every array where it has
// none at all), to be left out by `in`.
struct Edge {
  bool in;
  int e;       // CSR slot
  int64_t j;   // the other node
  __device__ Edge(const Item& it, int o, const int32_t* col) {
    in = o < it.n;
    e = it.n > 0 ? it.beg + (in ? o : 0) : 0;
    const int c = col[e];
    j = it.n > 0 ? c : 0;
  }
};
// Edges whose rows are in flight per slot. Logits: 8 of the 16-bit types (PPI, bf16 d = 128 / fp16 d =
// 64: 206 / 119 us, against 220 / 134 with 4), 4 of float32 (d = 61: 318 us, 373 with 8). The other
// passes keep more waves with 2 (fp16: values 103 us, 112 with 4; dw 98 / 108; gq 118 / 128).
template <typename T>
constexpr int kDotFlight = sizeof(T) == 2 ? 8 : 4;
constexpr int kFlight = 2;

// One row's state over a slot's edges: both maps' running maximum and sum.
template <int NV>
struct Acc {
  float m1 = -kInf, m2 = -kInf, l1 = 0.f, l2 = 0.f;
  float a1[NV][8] = {}, a2[NV][8] = {};
};
__device__ inline float finite_max(float m) { return m == -kInf ? 0.f : m; }
// {max, 1 / sum} of both maps; nothing open: weights of 0
__device__ inline float4 row_stat(float m1, float s1, float m2, float s2) {
  return make_float4(finite_max(m1), s1 == 0.f ? 0.f : 1.f / s1, finite_max(m2),
                     s2 == 0.f ? 0.f : 1.f / s2);
}

// U edges of a slot. CHECK: some lane of the wave has an edge that is past its row's end or shut;
// what such an edge points at is not let into the sums.
template <typename T, int G, int NV, int U, bool BIAS, bool CHECK>
__device__ inline void serve_step(const Raw<T> (&k1)[U], const Raw<T> (&k2)[U],
                                    const Raw<T> (&v)[U][NV], const Raw<T>& q1, const Raw<T>& q2,
                                    const float (&b)[U], const bool (&open)[U], bool in_d,
                                    float scale, Acc<NV>& acc) {
  float2 x[U];
  float n1 = acc.m1, n2 = acc.m2;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float s1 = dot8(q1, k1[u], 0.f), s2 = dot8(q2, k2[u], 0.f);
    x[u].x = edge_sum<G>(in_d ? s1 : 0.f) * scale;
    x[u].y = edge_sum<G>(in_d ? s2 : 0.f) * scale;
    if (BIAS) {
      x[u].x += b[u];
      x[u].y += b[u];
    }
    if (CHECK) {
      x[u].x = open[u] ? x[u].x : -kInf;
      x[u].y = open[u] ? x[u].y : -kInf;
    }
    n1 = fmaxf(n1, x[u].x);
    n2 = fmaxf(n2, x[u].y);
  }
  const float r1 = finite_max(n1), r2 = finite_max(n2);
  const float c1 = exp_(acc.m1 - r1), c2 = exp_(acc.m2 - r2);
  acc.m1 = n1;
  acc.m2 = n2;
  acc.l1 *= c1;
  acc.l2 *= c2;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc.a1[j][i] *= c1;
      acc.a2[j][i] *= c2;
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float p1 = exp_(x[u].x - r1), p2 = exp_(x[u].y - r2);
    acc.l1 += p1;
    acc.l2 += p2;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[8];
      unpack8(CHECK ? keep8(open[u], v[u][j]) : v[u][j], f);
      axpy8(p1, f, acc.a1[j]);
      axpy8(p2, f, acc.a2[j]);
    }
  }
}

// The serving form: one pass with running maxima and sums, each slot its own edges. Rows of k and v
// as they come (any alignment, d and dv of 8 or more): packing every node's for a few rows would be
// most of the call (70 000 nodes, 8 heads of d = 61, dv = 121 in bf16: about 110 us, the call itself
// 9 us for 30 edges and 61 us for 65 537). The last chunk of a row then starts early enough to end
// with it; what it shares with the chunk before is left out of q and k, and stored twice alike of
// the values.
template <typename T, int G, int NV, bool BIAS>
__global__ void __launch_bounds__(256) diff_serve_kernel(AttnArgs a) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;
  const Item it = find_item(a.w);
  Lane<G, NV> l(a.w.gs, a.dp, a.dvp);
  const int wd = a.kv_plain ? a.d : a.dp, wv = a.kv_plain ? a.dv : a.dvp;
  const int chunk = l.at_d;
  l.at_d = min(l.at_d, wd - 8);
#pragma unroll
  for (int i = 0; i < NV; ++i) l.at_dv[i] = min(l.at_dv[i], wv - 8);
  const From<T> own(chunk - l.at_d);
  const bool has = it.row >= 0;
  const int64_t row = has ? it.row : 0;
  const Raw<T> q1 = own(load_q<T>(a, row, it.head, 0, l.at_d));
  const Raw<T> q2 = own(load_q<T>(a, row, it.head, 1, l.at_d));
  Acc<NV> acc;
  const T* kb = (const T*)a.k + (int64_t)it.head * 2 * wd + l.at_d;
  const T* vb = (const T*)a.v + (int64_t)it.head * wv;
  const int turns = turns_of(wave_max(it.n), l.slots * U);
  for (int t = 0; t < turns; ++t) {
    Raw<T> k1[U], k2[U], v[U][NV];
    float b[U];
    bool open[U], all = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Edge e(it, (t * U + u) * l.slots + l.slot, a.col);
      open[u] = e.in;
      b[u] = 0.f;
      if (BIAS) {
        const int bk = a.bucket[e.e];   // (past the end: not necessarily one)
        b[u] = a.bias[(e.in ? bk : 0) * a.w.heads + it.head];
        open[u] = open[u] && b[u] != -kInf;
      }
      all = all && open[u];
      k1[u] = load8_anywhere(kb + e.j * a.ldk);
      k2[u] = load8_anywhere(kb + e.j * a.ldk + wd);
#pragma unroll
      for (int i = 0; i < NV; ++i) v[u][i] = load8_anywhere(vb + e.j * a.ldv + l.at_dv[i]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k1[u] = own(k1[u]);
      k2[u] = own(k2[u]);
    }
    if (__all(all))
      serve_step<T, G, NV, U, BIAS, false>(k1, k2, v, q1, q2, b, open, l.in_d, a.scale, acc);
    else
      serve_step<T, G, NV, U, BIAS, true>(k1, k2, v, q1, q2, b, open, l.in_d, a.scale, acc);
  }
  // the slots joined
  const int c = l.c, slot = l.slot;
  const float m1 = slots_max<G>(acc.m1, a.w.gs), m2 = slots_max<G>(acc.m2, a.w.gs);
  const float c1 = exp_(acc.m1 - finite_max(m1)), c2 = exp_(acc.m2 - finite_max(m2));
  float ls[2] = {acc.l1 * c1, acc.l2 * c2};
  slots_sum<G>(ls, a.w.gs);
  const float l1 = ls[0], l2 = ls[1];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc.a1[j][i] *= c1;
      acc.a2[j][i] *= c2;
    }
    slots_sum<G>(acc.a1[j], a.w.gs);
    slots_sum<G>(acc.a2[j], a.w.gs);
  }
  if (!has || slot != 0) return;
  // where the chunks go: past the end there is nothing to write but what a plain row's last has
  int at[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) at[j] = a.kv_plain ? l.at_dv[j] : (c + j * G) * 8;
  const bool whole = a.dv == a.dvp;
  if (it.slot >= 0) {   // a piece: {m1, l1, m2, l2, sums of map 1, of map 2}
    float* p = a.part + ((int64_t)it.slot * a.w.heads + it.head) * a.part_width;
    if (c == 0) *(float4*)p = make_float4(m1, it.bad ? __builtin_nanf("") : l1, m2, l2);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      store8(p + 4, at[j], a.dvp, whole, acc.a1[j]);
      store8(p + 4 + a.dvp, at[j], a.dvp, whole, acc.a2[j]);
    }
    return;
  }
  const float i1 = l1 == 0.f ? 0.f : 1.f / l1, i2 = l2 == 0.f ? 0.f : 1.f / l2;
  const float w2 = a.lam[it.head] * i2;
  T* out = (T*)a.out + (row * a.w.heads + it.head) * a.dv;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = acc.a1[j][i] * i1 - acc.a2[j][i] * w2;
      if (it.bad) o[i] = __builtin_nanf("");
    }
    store8(out, at[j], a.dv, whole, o);
  }
}

// The pieces of a served row joined: a workgroup per (row, head, 32 columns), both maps' sums in 16
// runs of pieces side by side, each run and then the runs in order. (One node of 65 537 edges, 8
// heads in 256 pieces: 14 us with a workgroup per (row, head).)
constexpr int kJoinCols = 32, kJoinRuns = 16;
template <typename T>
__global__ void __launch_bounds__(1024) diff_serve_join_kernel(AttnArgs a) {
  __shared__ float sums[kJoinRuns][2 * kJoinCols];
  const int cb = (a.dv + kJoinCols - 1) / kJoinCols;
  const int64_t rh = blockIdx.x / cb, row = rh / a.w.heads;
  const int x0 = (int)(blockIdx.x - rh * cb) * kJoinCols;
  const int head = (int)(rh - row * a.w.heads), pieces = a.w.pieces, H = a.w.heads;
  const float* p0 = a.part + (row * pieces * H + head) * a.part_width;
  const int64_t step = (int64_t)H * a.part_width;
  // every wave finds the maxima and sums for itself
  const int lane = threadIdx.x & 63;
  float m1 = -kInf, m2 = -kInf, l1 = 0.f, l2 = 0.f;
  for (int i = lane; i < pieces; i += 64) {
    const float4 s = *(const float4*)(p0 + i * step);
    const float n1 = fmaxf(m1, s.x), n2 = fmaxf(m2, s.z);
    const float r1 = finite_max(n1), r2 = finite_max(n2);
    l1 = l1 * exp_(m1 - r1) + s.y * exp_(s.x - r1);
    l2 = l2 * exp_(m2 - r2) + s.w * exp_(s.z - r2);
    m1 = n1;
    m2 = n2;
  }
  const float t1 = slots_max<1>(m1, 64), t2 = slots_max<1>(m2, 64);
  const float r1 = finite_max(t1), r2 = finite_max(t2);
  l1 = group_sum<64>(l1 * exp_(m1 - r1));
  l2 = group_sum<64>(l2 * exp_(m2 - r2));
  // thread: column (lane & 31) of map (lane >> 5), run = its wave
  const int run = threadIdx.x >> 6, x = x0 + (lane & 31), map = lane >> 5;
  const float r = map ? r2 : r1;
  float s = 0.f;
  if (x < a.dv) {
    const float* p = p0 + 4 + map * a.dvp + x;
#pragma unroll 4
    for (int i = run; i < pieces; i += kJoinRuns)
      s += p[i * step] * exp_(p0[i * step + 2 * map] - r);
  }
  sums[run][lane] = s;
  __syncthreads();
  if (run != 0 || map != 0 || x >= a.dv) return;
  float s1 = 0.f, s2 = 0.f;
  for (int k = 0; k < kJoinRuns; ++k) {
    s1 += sums[k][lane];
    s2 += sums[k][kJoinCols + lane];
  }
  const float i1 = l1 == 0.f ? 0.f : 1.f / l1, i2 = l2 == 0.f ? 0.f : 1.f / l2;
  ((T*)a.out)[(row * H + head) * a.dv + x] = (T)(s1 * i1 - s2 * (a.lam[head] * i2));
}

// ------------------------------------------------------------------ forward over whole rows
// Both maps' weights of an edge from its logits; a shut or -inf logit has weight 0 whatever the
// statistics hold.
__device__ inline float2 weights(float2 x, const float4& st) {
  return make_float2(x.x == -kInf ? 0.f : exp_(x.x - st.x) * st.y,
                     x.y == -kInf ? 0.f : exp_(x.y - st.z) * st.w);
}

// An item's pass over its edges in tiles: `first` of a tile's first edge in this slot, turn by turn.
template <int G>
struct Tiles {
  int lane, mine, step, most;   // mine: the edge of a tile this lane holds
  bool owner;                   // (of G = 32 lanes the second 16 hold the first's edges again)
  __device__ Tiles(const Item& it, int gs) {
    lane = threadIdx.x & 63;
    mine = lane & (kTile<G> - 1);
    owner = G < 32 || (lane & 31) < 16;
    step = gs / G * kTile<G>;
    most = wave_max(it.n);
  }
  __device__ int first(int t, int slot) const { return t * step + slot * kTile<G>; }
  // no lane of the wave has an edge from number i of its tile on
  __device__ bool done(int t, int i) const { return t * step + i >= most; }
};

// The logits of every edge and the softmax statistics of every row.
template <typename T, int G, bool BIAS>
__global__ void __launch_bounds__(256) diff_score_kernel(AttnArgs a) {
  constexpr int NL = kTile<G>, U = NL < kDotFlight<T> ? NL : kDotFlight<T>;
  const Item it = find_item(a.w);
  const Lane<G, 1> l(a.w.gs, a.dp, 8);
  const Tiles<G> tl(it, a.w.gs);
  const bool has = it.row >= 0;
  const int64_t row = has ? it.row : 0;
  const Raw<T> q1 = load_q<T>(a, row, it.head, 0, l.at_d), q2 = load_q<T>(a, row, it.head, 1, l.at_d);
  const T* kb = (const T*)a.k + (int64_t)it.head * 2 * a.dp + l.at_d;
  const int64_t he = (int64_t)it.head * a.E;
  float m1 = -kInf, m2 = -kInf, s1 = 0.f, s2 = 0.f;
  for (int t = 0; !tl.done(t, 0); ++t) {
    const int o = tl.first(t, l.slot) + tl.mine;
    const Edge e(it, o, a.col);
    const int64_t off = row_off<T>(e.j, a.ldk);
    float b = 0.f;
    if (BIAS) {
      const int bk = a.bucket[e.e];   // (past the end: not necessarily one)
      b = a.bias[(e.in ? bk : 0) * a.w.heads + it.head];
    }
    float x1[NL], x2[NL];
    each<NL / U>([&](auto B) {
      constexpr int b0 = decltype(B)::value * U;
      if (b0 > 0 && tl.done(t, b0)) {
#pragma unroll
        for (int u = 0; u < U; ++u) x1[b0 + u] = x2[b0 + u] = 0.f;
        return;
      }
      Raw<T> k1[U], k2[U];
      each<U>([&](auto I) {
        constexpr int u = decltype(I)::value;
        const T* p = row_at(kb, tile_get<G, b0 + u>(off));
        k1[u] = load8(p);
        k2[u] = load8(p + a.dp);
      });
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float d1 = dot8(q1, k1[u], 0.f), d2 = dot8(q2, k2[u], 0.f);
        x1[b0 + u] = l.in_d ? d1 : 0.f;
        x2[b0 + u] = l.in_d ? d2 : 0.f;
      }
    });
    float2 x;
    x.x = fmaf(tile_scatter<G>(x1, tl.lane), a.scale, b);
    x.y = fmaf(tile_scatter<G>(x2, tl.lane), a.scale, b);
    const bool shut = !e.in || (BIAS && b == -kInf);
    x.x = shut ? -kInf : x.x;
    x.y = shut ? -kInf : x.y;
    if (tl.owner) {
      if (e.in) a.S[he + e.e] = x;
      const float n1 = fmaxf(m1, x.x), n2 = fmaxf(m2, x.y);
      const float r1 = finite_max(n1), r2 = finite_max(n2);
      s1 = s1 * exp_(m1 - r1) + exp_(x.x - r1);
      s2 = s2 * exp_(m2 - r2) + exp_(x.y - r2);
      m1 = n1;
      m2 = n2;
    }
  }
  // the lanes joined
  const float t1 = slots_max<1>(m1, a.w.gs), t2 = slots_max<1>(m2, a.w.gs);
  float s[2] = {s1 * exp_(m1 - finite_max(t1)), s2 * exp_(m2 - finite_max(t2))};
  slots_sum<1>(s, a.w.gs);
  if (!has || l.c != 0 || l.slot != 0) return;
  if (it.slot >= 0)
    *(float4*)(a.part + ((int64_t)it.slot * a.w.heads + it.head) * 4) =
        make_float4(t1, s[0], t2, s[1]);
  else
    a.stat[(int64_t)it.head * a.w.rows + row] = row_stat(t1, s[0], t2, s[1]);
}

// out of every row: its values weighted by p_1 - lam p_2.
template <typename T, int G, int NV>
__global__ void __launch_bounds__(256) diff_value_kernel(AttnArgs a) {
  constexpr int NL = kTile<G>, U = NL < kFlight ? NL : kFlight;
  const Item it = find_item(a.w);
  const Lane<G, NV> l(a.w.gs, a.dp, a.dvp);
  const Tiles<G> tl(it, a.w.gs);
  const bool has = it.row >= 0;
  const int64_t row = has ? it.row : 0;
  const float4 st = a.stat[(int64_t)it.head * a.w.rows + row];
  const float lam = a.lam[it.head];
  const T* vb = (const T*)a.v + (int64_t)it.head * a.dvp;
  const int64_t he = (int64_t)it.head * a.E;
  float acc[NV][8] = {};
  for (int t = 0; !tl.done(t, 0); ++t) {
    const Edge e(it, tl.first(t, l.slot) + tl.mine, a.col);
    const int64_t off = row_off<T>(e.j, a.ldv);
    const float2 x = a.S[he + e.e], p = weights(x, st);
    const bool open = e.in && (x.x != -kInf || x.y != -kInf);
    const Keep<T> keep(open);
    const float w = open ? p.x - lam * p.y : 0.f;
    auto edges = [&](auto ALL) {
      each<NL / U>([&](auto B) {
        constexpr int b0 = decltype(B)::value * U;
        if (b0 > 0 && tl.done(t, b0)) return;
        Raw<T> v[U][NV];
        each<U>([&](auto I) {
          constexpr int u = decltype(I)::value;
          const T* p = row_at(vb, tile_get<G, b0 + u>(off));
#pragma unroll
          for (int i = 0; i < NV; ++i) v[u][i] = load8(p + l.at_dv[i]);
        });
        each<U>([&](auto I) {
          constexpr int u = decltype(I)::value;
          const float wu = tile_get<G, b0 + u>(w);
          const Keep<T> ku = keep.template of_edge<G, b0 + u>();
#pragma unroll
          for (int i = 0; i < NV; ++i) axpy_kept<decltype(ALL)::value>(wu, v[u][i], ku, acc[i]);
        });
      });
    };
    if (__all(open)) edges(std::true_type());
    else edges(std::false_type());
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) slots_sum<G>(acc[i], a.w.gs);
  if (!has || l.slot != 0) return;
  if (it.slot >= 0) {
    float* p = a.part + ((int64_t)it.slot * a.w.heads + it.head) * a.part_width;
#pragma unroll
    for (int i = 0; i < NV; ++i) store8(p, (l.c + i * G) * 8, a.dvp, true, acc[i]);
    return;
  }
  T* out = (T*)a.out + (row * a.w.heads + it.head) * a.dv;
#pragma unroll
  for (int i = 0; i < NV; ++i) store8(out, (l.c + i * G) * 8, a.dv, a.dv == a.dvp, acc[i]);
}

// The hubs of the plan, in a fixed grid of workgroups: f(first slot, node, pieces, head).
template <typename F>
__device__ inline void each_hub(const Work& w, int64_t at, int64_t step, F&& f) {
  const int64_t n = (int64_t)min(*w.hub_count, w.hub_bound) * w.heads;
  for (int64_t i = at; i < n; i += step) {
    const int pc = (int)(i / w.heads);
    const int32_t* hp = w.hubs + 4 * (int64_t)pc;
    if (hp[1] == 0) f(pc, hp[0], hp[2], (int)(i - (int64_t)pc * w.heads));   // its first entry
  }
}
// Statistics of the hubs from their pieces'.
__global__ void __launch_bounds__(256) diff_score_join_kernel(AttnArgs a) {
  each_hub(a.w, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256,
           [&](int first, int row, int pieces, int head) {
             auto part = [&](int k) {
               return *(const float4*)(a.part + ((int64_t)(first + k) * a.w.heads + head) * 4);
             };
             float m1 = -kInf, m2 = -kInf, s1 = 0.f, s2 = 0.f;
             for (int k = 0; k < pieces; ++k) {
               m1 = fmaxf(m1, part(k).x);
               m2 = fmaxf(m2, part(k).z);
             }
             for (int k = 0; k < pieces; ++k) {
               s1 += part(k).y * exp_(part(k).x - finite_max(m1));
               s2 += part(k).w * exp_(part(k).z - finite_max(m2));
             }
             a.stat[(int64_t)head * a.w.rows + row] = row_stat(m1, s1, m2, s2);
           });
}
// Sums of the hubs' pieces: [two maps of dp (where maps_in) | dvp] columns, a thread a column.
template <typename T>
__global__ void __launch_bounds__(256) diff_sum_join_kernel(AttnArgs a, int maps_in, T* maps,
                                                            T* values) {
  const int W = a.part_width, dp2 = maps_in ? 2 * a.dp : 0;
  each_hub(a.w, blockIdx.x, gridDim.x, [&](int first, int row, int pieces, int head) {
    const int64_t rh = (int64_t)row * a.w.heads + head, step = (int64_t)a.w.heads * W;
    for (int x = threadIdx.x; x < W; x += 256) {
      const float* p = a.part + ((int64_t)first * a.w.heads + head) * W + x;
      float s = 0.f;
#pragma unroll 8
      for (int k = 0; k < pieces; ++k) s += p[k * step];
      if (x < dp2) {
        const int m = x >= a.dp, y = x - m * a.dp;
        if (maps && y < a.d) maps[(rh * 2 + m) * a.d + y] = (T)s;
      } else if (values && x - dp2 < a.dv) {
        values[rh * a.dv + x - dp2] = (T)s;
      }
    }
  });
}

// ------------------------------------------------------------------ backward
// A: dw = go . v of every edge, D_1 and D_2 of every row.
template <typename T, int G, int NV>
__global__ void __launch_bounds__(256) diff_dw_kernel(AttnArgs a) {
  constexpr int NL = kTile<G>, U = NL < kFlight ? NL : kFlight;
  const Item it = find_item(a.w);
  const Lane<G, NV> l(a.w.gs, a.dp, a.dvp);
  const Tiles<G> tl(it, a.w.gs);
  const bool has = it.row >= 0;
  const int64_t row = has ? it.row : 0;
  const T* gr = (const T*)a.go + row * a.ldgo + (int64_t)it.head * a.dvp;
  Raw<T> g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) g[i] = load8(gr + l.at_dv[i]);
  const float4 st = a.stat[(int64_t)it.head * a.w.rows + row];
  const T* vb = (const T*)a.v + (int64_t)it.head * a.dvp;
  const int64_t he = (int64_t)it.head * a.E;
  float d[2] = {0.f, 0.f};
  for (int t = 0; !tl.done(t, 0); ++t) {
    const Edge e(it, tl.first(t, l.slot) + tl.mine, a.col);
    const int64_t off = row_off<T>(e.j, a.ldv);
    const float2 x = a.S[he + e.e];
    float y[NL];
    each<NL / U>([&](auto B) {
      constexpr int b0 = decltype(B)::value * U;
      if (b0 > 0 && tl.done(t, b0)) {
#pragma unroll
        for (int u = 0; u < U; ++u) y[b0 + u] = 0.f;
        return;
      }
      Raw<T> v[U][NV];
      each<U>([&](auto I) {
        constexpr int u = decltype(I)::value;
        const T* p = row_at(vb, tile_get<G, b0 + u>(off));
#pragma unroll
        for (int i = 0; i < NV; ++i) v[u][i] = load8(p + l.at_dv[i]);
      });
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float p = dot8(g[i], v[u][i], 0.f);
          s += l.in_dv[i] ? p : 0.f;
        }
        y[b0 + u] = s;
      }
    });
    float dw = tile_scatter<G>(y, tl.lane);
    if (x.x == -kInf && x.y == -kInf) dw = 0.f;   // shut: its value does not count
    if (e.in && tl.owner) {
      const float2 p = weights(x, st);
      d[0] = fmaf(p.x, dw, d[0]);
      d[1] = fmaf(p.y, dw, d[1]);
      a.dw[he + e.e] = dw;
    }
  }
  slots_sum<1>(d, a.w.gs);
  if (!has || l.c != 0 || l.slot != 0) return;
  if (it.slot >= 0)
    *(float2*)(a.part + ((int64_t)it.slot * a.w.heads + it.head) * 2) = make_float2(d[0], d[1]);
  else
    a.D[(int64_t)it.head * a.w.rows + row] = make_float2(d[0], d[1]);
}
__global__ void __launch_bounds__(256) diff_dw_join_kernel(AttnArgs a) {
  each_hub(a.w, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256,
           [&](int first, int row, int pieces, int head) {
             float2 d = make_float2(0.f, 0.f);
             for (int k = 0; k < pieces; ++k) {
               const float2 p =
                   *(const float2*)(a.part + ((int64_t)(first + k) * a.w.heads + head) * 2);
               d.x += p.x;
               d.y += p.y;
             }
             a.D[(int64_t)head * a.w.rows + row] = d;
           });
}

// B: gq of every row, and each edge's record for C and the bias.
template <typename T, int G>
__global__ void __launch_bounds__(256) diff_gq_kernel(AttnArgs a) {
  constexpr int NL = kTile<G>, U = NL < kFlight ? NL : kFlight;
  const Item it = find_item(a.w);
  const Lane<G, 1> l(a.w.gs, a.dp, 8);
  const Tiles<G> tl(it, a.w.gs);
  const bool has = it.row >= 0;
  const int64_t row = has ? it.row : 0, sr = (int64_t)it.head * a.w.rows + row;
  const float4 st = a.stat[sr];
  const float2 D = a.D[sr];
  const float lam = a.lam[it.head];
  const T* kb = (const T*)a.k + (int64_t)it.head * 2 * a.dp + l.at_d, *kb2 = kb + a.dp;
  const int64_t he = (int64_t)it.head * a.E;
  float g1[8] = {}, g2[8] = {};
  for (int t = 0; !tl.done(t, 0); ++t) {
    const Edge e(it, tl.first(t, l.slot) + tl.mine, a.col);
    const int64_t off = row_off<T>(e.j, a.ldk);
    const float2 x = a.S[he + e.e], p = weights(x, st);
    const float dw = a.dw[he + e.e];
    const bool open = e.in && (x.x != -kInf || x.y != -kInf);
    const Keep<T> keep(open);
    const float x1 = open ? p.x * (dw - D.x) : 0.f;
    const float x2 = open ? -lam * p.y * (dw - D.y) : 0.f;
    if (e.in && tl.owner)
      a.rec[he + e.e] = make_float4(x1 * a.scale, x2 * a.scale, open ? p.x - lam * p.y : 0.f,
                                    x1 + x2);
    if (!a.gq) continue;
    auto edges = [&](auto ALL) {
      each<NL / U>([&](auto B) {
        constexpr int b0 = decltype(B)::value * U;
        if (b0 > 0 && tl.done(t, b0)) return;
        Raw<T> k1[U], k2[U];
        each<U>([&](auto I) {
          constexpr int u = decltype(I)::value;
          const int64_t at = tile_get<G, b0 + u>(off);
          k1[u] = load8(row_at(kb, at));
          k2[u] = load8(row_at(kb2, at));
        });
        each<U>([&](auto I) {
          constexpr int u = decltype(I)::value;
          const float y1 = tile_get<G, b0 + u>(x1), y2 = tile_get<G, b0 + u>(x2);
          const Keep<T> ku = keep.template of_edge<G, b0 + u>();
          axpy_kept<decltype(ALL)::value>(y1, k1[u], ku, g1);
          axpy_kept<decltype(ALL)::value>(y2, k2[u], ku, g2);
        });
      });
    };
    if (__all(open)) edges(std::true_type());
    else edges(std::false_type());
  }
  slots_sum<G>(g1, a.w.gs);
  slots_sum<G>(g2, a.w.gs);
  if (!has || l.slot != 0 || !a.gq) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    g1[i] *= a.scale;
    g2[i] *= a.scale;
  }
  if (it.slot >= 0) {
    float* p = a.part + ((int64_t)it.slot * a.w.heads + it.head) * a.part_width;
    store8(p, l.c * 8, a.dp, true, g1);
    store8(p + a.dp, l.c * 8, a.dp, true, g2);
  } else {
    T* gq = (T*)a.gq + (row * a.w.heads + it.head) * 2 * a.d;
    store8(gq, l.c * 8, a.d, a.d == a.dp, g1);
    store8(gq + a.d, l.c * 8, a.d, a.d == a.dp, g2);
  }
}

// C: gk and gv of every source from its out-edges (CSR w.rowptr = srowptr, col = scol).
template <typename T, int G, int NV>
__global__ void __launch_bounds__(256) diff_gkv_kernel(AttnArgs a) {
  constexpr int NL = kTile<G>, U = NL < kFlight ? NL : kFlight;
  const Item it = find_item(a.w);
  const Lane<G, NV> l(a.w.gs, a.dp, a.dvp);
  const Tiles<G> tl(it, a.w.gs);
  const bool has = it.row >= 0;
  const int64_t row = has ? it.row : 0;
  const T* qb = (const T*)a.q + (int64_t)it.head * 2 * a.dp + l.at_d, *qb2 = qb + a.dp;
  const T* gb[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) gb[k] = (const T*)a.go + (int64_t)it.head * a.dvp + l.at_dv[k];
  const float4* rec = a.rec + (int64_t)it.head * a.E;
  float g1[8] = {}, g2[8] = {}, gv[NV][8] = {};
  for (int t = 0; !tl.done(t, 0); ++t) {
    const Edge e(it, tl.first(t, l.slot) + tl.mine, a.col);
    const int64_t offq = row_off<T>(e.j, a.ldq), offg = row_off<T>(e.j, a.ldgo);
    const int id = a.seid[e.e];
    const float4 r = rec[it.n > 0 ? id : 0];
    // a shut edge is all zeros: what it points at does not count
    const bool open = e.in && (r.x != 0.f || r.y != 0.f || r.z != 0.f);
    const Keep<T> keep(open);
    const float r1 = open ? r.x : 0.f, r2 = open ? r.y : 0.f, rw = open ? r.z : 0.f;
    auto edges = [&](auto ALL) {
      each<NL / U>([&](auto B) {
        constexpr int b0 = decltype(B)::value * U;
        if (b0 > 0 && tl.done(t, b0)) return;
        Raw<T> q1[U], q2[U], go[U][NV];
        each<U>([&](auto I) {
          constexpr int u = decltype(I)::value;
          const int64_t at = tile_get<G, b0 + u>(offq), atg = tile_get<G, b0 + u>(offg);
          q1[u] = load8(row_at(qb, at));
          q2[u] = load8(row_at(qb2, at));
#pragma unroll
          for (int k = 0; k < NV; ++k) go[u][k] = load8(row_at(gb[k], atg));
        });
        each<U>([&](auto I) {
          constexpr int u = decltype(I)::value;
          constexpr bool all = decltype(ALL)::value;
          const Keep<T> ku = keep.template of_edge<G, b0 + u>();
          const float w1 = tile_get<G, b0 + u>(r1), w2 = tile_get<G, b0 + u>(r2),
                      w = tile_get<G, b0 + u>(rw);
          axpy_kept<all>(w1, q1[u], ku, g1);
          axpy_kept<all>(w2, q2[u], ku, g2);
#pragma unroll
          for (int k = 0; k < NV; ++k) axpy_kept<all>(w, go[u][k], ku, gv[k]);
        });
      });
    };
    if (__all(open)) edges(std::true_type());
    else edges(std::false_type());
  }
  slots_sum<G>(g1, a.w.gs);
  slots_sum<G>(g2, a.w.gs);
#pragma unroll
  for (int k = 0; k < NV; ++k) slots_sum<G>(gv[k], a.w.gs);
  if (!has || l.slot != 0) return;
  const int c = l.c;
  if (it.slot >= 0) {
    float* p = a.part + ((int64_t)it.slot * a.w.heads + it.head) * a.part_width;
    store8(p, c * 8, a.dp, true, g1);
    store8(p + a.dp, c * 8, a.dp, true, g2);
#pragma unroll
    for (int k = 0; k < NV; ++k) store8(p + 2 * a.dp, (c + k * G) * 8, a.dvp, true, gv[k]);
    return;
  }
  const int64_t rh = row * a.w.heads + it.head;
  if (a.gk) {
    T* gk = (T*)a.gk + rh * 2 * a.d;
    store8(gk, c * 8, a.d, a.d == a.dp, g1);
    store8(gk + a.d, c * 8, a.d, a.d == a.dp, g2);
  }
  if (a.gv) {
    T* out = (T*)a.gv + rh * a.dv;
#pragma unroll
    for (int k = 0; k < NV; ++k) store8(out, (c + k * G) * 8, a.dv, a.dv == a.dvp, gv[k]);
  }
}

// glam[h] = -sum of D_2 over the rows: a workgroup per (run of rows, head), then the runs in order.
// In float64: the rows' D_2 have both signs, and their sum is far smaller than they are together.
constexpr int kLamRuns = 64;
__global__ void __launch_bounds__(256) diff_lam_kernel(const float2* D, int64_t rows, int64_t per,
                                                       double* part, float* glam) {
  __shared__ double red[256];
  const int h = blockIdx.y;
  const int64_t r0 = blockIdx.x * per, r1 = min(rows, r0 + per);
  double s = 0.0;
#pragma unroll 4
  for (int64_t r = r0 + threadIdx.x; r < r1; r += 256) s += (double)D[h * rows + r].y;
  red[threadIdx.x] = s;
  for (int d = 128; d > 0; d >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
  }
  if (threadIdx.x) return;
  if (gridDim.x == 1) glam[h] = (float)-red[0];
  else part[h * gridDim.x + blockIdx.x] = red[0];
}
__global__ void __launch_bounds__(64) diff_lam_join_kernel(const double* part, int runs, int heads,
                                                           float* glam) {
  const int h = blockIdx.x * 64 + threadIdx.x;
  if (h >= heads) return;
  double s = 0.0;
#pragma unroll 8
  for (int i = 0; i < runs; ++i) s += part[h * runs + i];
  glam[h] = (float)-s;
}

// gbias: each lane adds its edges' dx_1 + dx_2 into a column of its own of an LDS table [bucket]
// [lane] (no two lanes share a word, so no atomics and one order), a wave per run of slots of one
// head; the lanes' columns, then the runs, are summed in order.
__global__ void __launch_bounds__(64) diff_bias_kernel(const float4* rec, const uint8_t* bucket,
                                                       const int32_t* rowptr, int64_t num_nodes,
                                                       int64_t E, int64_t per, int nb,
                                                       float* part) {
  extern __shared__ float hist[];   // [nb][64]
  const int lane = threadIdx.x, h = blockIdx.y;
  for (int b = 0; b < nb; ++b) hist[b * 64 + lane] = 0.f;
  const int64_t end = min((int64_t)rowptr[num_nodes], (int64_t)(blockIdx.x + 1) * per);
  const float* r = (const float*)(rec + h * E) + 3;
  int64_t e = blockIdx.x * per + lane;
  for (; e + 192 < end; e += 256) {
    float x[4];
    int b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x[u] = r[4 * (e + 64 * u)];
      b[u] = bucket[e + 64 * u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) hist[b[u] * 64 + lane] += x[u];
  }
  for (; e < end; e += 64) hist[(int)bucket[e] * 64 + lane] += r[4 * e];
  float* p = part + ((int64_t)h * gridDim.x + blockIdx.x) * nb;
  for (int b = 0; b < nb; ++b) {
    const float s = group_sum<64>(hist[b * 64 + lane]);
    if (lane == 0) p[b] = s;
  }
}
__global__ void __launch_bounds__(64) diff_bias_join_kernel(const float* part, int runs, int nb,
                                                            int heads, float* gbias) {
  const int b = blockIdx.x, h = blockIdx.y;
  float s = 0.f;
  for (int i = threadIdx.x; i < runs; i += 64) s += part[((int64_t)h * runs + i) * nb + b];
  s = group_sum<64>(s);
  if (threadIdx.x == 0) gbias[b * heads + h] = s;
}

// ------------------------------------------------------------------ buckets and packing
struct BucketArgs {
  const int32_t *rowptr, *col, *rowidx;
  const int64_t* nodes;
  int64_t num_nodes, n_nodes;
  const void* pos;
  int pos64, exact, n_bounds, bidirectional;
  int64_t bounds[kMaxBuckets / 2];
  uint8_t* bucket;
};
__device__ inline uint8_t bucket_of(const BucketArgs& a, const int64_t* bounds, int64_t src,
                                    int64_t dst) {
  auto at = [&](int64_t n) {
    return a.pos64 ? ((const int64_t*)a.pos)[n] : (int64_t)((const int32_t*)a.pos)[n];
  };
  const int64_t s = at(src), d = at(dst);
  // as unsigned: the difference of any two int64 fits
  uint64_t away = s > d ? (uint64_t)s - (uint64_t)d : (uint64_t)d - (uint64_t)s;
  int b = 0;
  if (a.bidirectional) b = s > d ? a.exact + a.n_bounds + 1 : 0;
  else if (s > d) away = 0;
  if (away < (uint64_t)a.exact) return (uint8_t)(b + (int)away);
  int lo = 0, hi = a.n_bounds;   // the number of bounds <= away
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((uint64_t)bounds[mid] <= away) lo = mid + 1;
    else hi = mid;
  }
  return (uint8_t)(b + a.exact + lo);
}
// One thread a slot; with nodes, a workgroup row of the grid walks one node's slots.
__global__ void __launch_bounds__(256) relative_bucket_kernel(BucketArgs a) {
  __shared__ int64_t bounds[kMaxBuckets / 2];
  if ((int)threadIdx.x < a.n_bounds) bounds[threadIdx.x] = a.bounds[threadIdx.x];
  __syncthreads();
  if (!a.nodes) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e < a.rowptr[a.num_nodes]) a.bucket[e] = bucket_of(a, bounds, a.col[e], a.rowidx[e]);
    return;
  }
  for (int64_t i = blockIdx.y; i < a.n_nodes; i += gridDim.y) {
    const int64_t n = a.nodes[i];
    if (n < 0 || n >= a.num_nodes) continue;
    const int end = a.rowptr[n + 1];
    for (int64_t e = (int64_t)a.rowptr[n] + blockIdx.x * 256 + threadIdx.x; e < end;
         e += (int64_t)gridDim.x * 256)
      a.bucket[e] = bucket_of(a, bounds, a.col[e], n);
  }
}

struct PackArgs {
  const void* src[3];
  void* dst[3];
  int64_t ld[3], n[3];   // n: elements of the packed tensor
  int groups[3], width[3], padded[3];
};
// Four bytes of the packed side a lane and round, four rounds in flight: both sides are read and
// written in order. (44 900 x 6 heads of d = 61, dv = 121 in float32: k and v in 100 us = 5.3 TB/s.)
template <typename T>
__global__ void __launch_bounds__(256) pack_heads_kernel(PackArgs a) {
  constexpr int R = 4, V = 4 / sizeof(T);
  const int t = blockIdx.y;
  const uint32_t w = a.width[t], wp = a.padded[t], row_elems = wp * a.groups[t];
  const int64_t i0 = ((int64_t)blockIdx.x * (256 * R) + threadIdx.x) * V;
  if (i0 >= a.n[t]) return;
  const T* src = (const T*)a.src[t];
  T* dst = (T*)a.dst[t];
  Pack<T, V> x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = min(i0 + r * 256 * V, a.n[t] - V), row = i / row_elems;
    const uint32_t in = (uint32_t)(i - row * row_elems), g = in / wp, c = in - g * wp;
    const T* p = src + row * a.ld[t] + g * w;
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) x[r].v[v] = p[min(c + v, w - 1)];
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) x[r].v[v] = c + v < w ? x[r].v[v] : (T)0.f;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = i0 + r * 256 * V;
    if (i < a.n[t]) *(Pack<T, V>*)(dst + i) = x[r];
  }
}

// ------------------------------------------------------------------ launches
struct Geom {
  int G, NV;
};
// The smallest G lanes that hold both maps' d in one chunk a lane and dv in at most two.
Geom attn_geom(int d, int dv) {
  const int dch = (int)ceil_div(d, 8), vch = (int)ceil_div(dv, 8);
  int G = 1;
  while (G < dch || 2 * G < vch) G <<= 1;
  return {G, vch > G ? 2 : 1};
}
template <typename F>
void with_geom(const Geom& g, F&& f) {
  auto nv = [&](auto G) {
    if (g.NV == 1) f(G, std::integral_constant<int, 1>());
    else f(G, std::integral_constant<int, 2>());
  };
  switch (g.G) {
    case 1: nv(std::integral_constant<int, 1>()); break;
    case 2: nv(std::integral_constant<int, 2>()); break;
    case 4: nv(std::integral_constant<int, 4>()); break;
    case 8: nv(std::integral_constant<int, 8>()); break;
    case 16: nv(std::integral_constant<int, 16>()); break;
    default: nv(std::integral_constant<int, 32>()); break;
  }
}
// Lanes of a row: as few as hold an edge (16 at least), so what a row costs once is spread over its
// edges and four rows share a wave; more where the rows alone would leave the chip short of waves.
int row_lanes(int G, int64_t items) {
  int gs = G > 16 ? G : 16;
  while (gs < 64 && items * gs < 64 * kWantWaves) gs <<= 1;
  return gs;
}

int log2i(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
// The plain rows' grid (and the pieces' blocks ahead of it).
int64_t plan_rows(Work& w, int64_t rows, int heads, int gs, const int32_t* rowptr,
                  const int32_t* order, int hub_edges, const int32_t* hubs,
                  const int32_t* hub_count, int64_t hub_bound) {
  w = Work{};
  w.rows = (int)rows;
  w.num_nodes = rows;
  w.heads = heads;
  w.gs = gs;
  w.gs_log = log2i(gs);
  w.rowptr = rowptr;
  w.order = gs < 64 ? (const int4*)order : nullptr;   // (a row to a wave: as they are)
  const int per_block = 256 / gs;
  // units of kChunk rows; fewer where that would leave XCDs without one
  const int64_t chunk = std::min<int64_t>(kChunk, ceil_div(rows * heads, 64));
  w.unit_log = log2i((int)ceil_div(chunk, per_block));
  const int64_t units = ceil_div(rows, (int64_t)per_block << w.unit_log) * heads;
  w.units = (int)std::min<int64_t>(units, INT32_MAX);
  if (hub_edges > 0 && hub_bound > 0) {
    w.hub_edges = hub_edges;
    w.hubs = hubs;
    w.hub_count = hub_count;
    w.hub_bound = (int)hub_bound;
    w.hub_blocks = (int)std::min<int64_t>(ceil_div(hub_bound * heads, per_block), INT32_MAX);
  }
  return w.hub_blocks + (round_up(units, 8) << w.unit_log);
}

int check_dims(const char* what, int dtype, int heads, int d, int dv, int64_t E, int64_t rows) {
  GATX_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
  GATX_REQUIRE(heads >= 1 && heads <= 65535, "%s: %d heads", what, heads);
  GATX_REQUIRE(d >= 1 && d <= kMaxD && dv >= 1 && dv <= kMaxDv,
               "%s: head widths d = %d (1..%d), dv = %d (1..%d)", what, d, kMaxD, dv, kMaxDv);
  GATX_REQUIRE(E >= 0 && E < (1ll << 31) && rows >= 0 && rows < (1ll << 31), "%s: bad graph size",
               what);
  return 0;
}
bool chunked(int dtype, const void* p, int64_t ld) {
  return aligned16(p) && ld * dtype_size(dtype) % 16 == 0;
}
// Workgroups of a join over the hubs, `per` (hub, head) pairs each: the plan's size is only bounded
// on the host, so a fixed number walks what there is.
unsigned join_blocks(const Work& w, int per) {
  return (unsigned)std::min<int64_t>(ceil_div((int64_t)w.hub_bound * w.heads, per), 1024);
}
// A launch holds fewer than 2^32 threads.
#define GATX_GRID(blocks, threads, what)                                                    \
  GATX_REQUIRE((blocks) * (threads) < (1ll << 32), "%s: too many work items for one launch", what)

}  // namespace
}  // namespace gatx

using namespace gatx;

extern "C" int gatx_relative_buckets(const int32_t* rowptr, const int32_t* col,
                                     const int32_t* rowidx, int64_t E, int64_t num_nodes,
                                     const int64_t* nodes, int64_t n_nodes, const void* pos,
                                     int pos_is64, int exact, const int64_t* bounds, int n_bounds,
                                     int bidirectional, uint8_t* bucket, gatx_stream_t s) {
  GATX_REQUIRE(exact >= 1 && n_bounds >= 0 && n_bounds < kMaxBuckets / 2 &&
               (exact + n_bounds + 1) * (bidirectional ? 2 : 1) <= kMaxBuckets,
               "relative_buckets: %d exact buckets and %d bounds (at most %d in all)", exact,
               n_bounds, kMaxBuckets);
  GATX_REQUIRE(n_bounds == 0 || bounds, "relative_buckets: null bounds");
  if (E == 0 || num_nodes == 0 || (nodes && n_nodes == 0)) return 0;
  GATX_REQUIRE(rowptr && col && pos && bucket && (nodes || rowidx),
               "relative_buckets: null buffer");
  BucketArgs a = {};
  a.rowptr = rowptr; a.col = col; a.rowidx = rowidx; a.nodes = nodes; a.num_nodes = num_nodes;
  a.n_nodes = n_nodes; a.pos = pos; a.pos64 = pos_is64; a.exact = exact; a.n_bounds = n_bounds;
  a.bidirectional = bidirectional; a.bucket = bucket;
  for (int i = 0; i < n_bounds; ++i) a.bounds[i] = bounds[i];
  dim3 grid((unsigned)ceil_div(E, 256));
  if (nodes)
    grid = dim3((unsigned)std::min<int64_t>(ceil_div(E, 256), std::max<int64_t>(1, 512 / n_nodes)),
                (unsigned)std::min<int64_t>(n_nodes, 32768));
  relative_bucket_kernel<<<grid, 256, 0, (hipStream_t)s>>>(a);
  GATX_LAUNCH_CHECK("relative_buckets");
  return 0;
}

extern "C" int gatx_diff_attention_pack(int dtype, int64_t rows, int64_t keys, int heads, int d,
                                        int dv, const void* q, int64_t ldq, void* qp,
                                        const void* k, int64_t ldk, void* kp, const void* v,
                                        int64_t ldv, void* vp, gatx_stream_t s) {
  GATX_CALL(check_dims("diff_attention_pack", dtype, heads, d, dv, 0, std::max(rows, keys)));
  PackArgs a = {};
  int t = 0;
  int64_t most = 0;
  auto add = [&](const void* src, int64_t ld, void* dst, int64_t n, int groups, int width) {
    if (!src || n == 0) return;
    a.src[t] = src; a.dst[t] = dst; a.ld[t] = ld; a.groups[t] = groups; a.width[t] = width;
    a.padded[t] = (int)round_up(width, 8);
    a.n[t] = n * groups * a.padded[t];
    most = std::max(most, a.n[t]);
    ++t;
  };
  add(q, ldq, qp, rows, 2 * heads, d);
  add(k, ldk, kp, keys, 2 * heads, d);
  add(v, ldv, vp, keys, heads, dv);
  if (t == 0) return 0;
  for (int i = 0; i < t; ++i)
    GATX_REQUIRE(a.dst[i] && aligned16(a.dst[i]), "diff_attention_pack: bad destination");
  const int64_t blocks = ceil_div(most * dtype_size(dtype), 4096);
  GATX_GRID(blocks, 256, "diff_attention_pack");
  const dim3 grid((unsigned)blocks, t);
  with_dtype(dtype, [&](auto x) {
    pack_heads_kernel<decltype(x)><<<grid, 256, 0, (hipStream_t)s>>>(a);
    return 0;
  });
  GATX_LAUNCH_CHECK("diff_attention_pack");
  return 0;
}

extern "C" int gatx_diff_attention_row_order(const int32_t* rowptr, int64_t rows, int32_t* order,
                                             gatx_stream_t s) {
  GATX_REQUIRE(rows >= 0 && rows < (1ll << 31), "diff_attention_row_order: bad graph size");
  if (rows == 0) return 0;
  GATX_REQUIRE(rowptr && order && aligned16(order), "diff_attention_row_order: null or unaligned");
  row_order_kernel<<<(unsigned)ceil_div(rows, kChunk), 64 * kOrderWaves, 0, (hipStream_t)s>>>(
      rowptr, rows, (int4*)order);
  GATX_LAUNCH_CHECK("diff_attention_row_order");
  return 0;
}

extern "C" size_t gatx_diff_attention_part_bytes(int64_t slots, int heads, int dvp) {
  return sizeof(float) * (size_t)std::max<int64_t>(slots, 0) * heads * (2 * dvp + 4);
}

extern "C" int gatx_diff_attention(int dtype, const void* q, int64_t ldq, const void* k,
                                   int64_t ldk, const void* v, int64_t ldv, int heads, int d,
                                   int dv, const int32_t* rowptr, const int32_t* col, int64_t E,
                                   int64_t rows, int64_t num_nodes, const int64_t* nodes,
                                   int pieces, float scale, const float* lam, const float* bias,
                                   const uint8_t* bucket, void* out, float* S, float* stat,
                                   int hub_edges, const int32_t* hubs, const int32_t* hub_count,
                                   int64_t hub_bound, void* part, size_t part_bytes,
                                   const int32_t* order, gatx_stream_t s) {
  const bool plain_q = dtype >= 0 && (dtype & GATX_Q_UNPACKED);
  const bool plain_kv = dtype >= 0 && (dtype & GATX_KV_UNPACKED);
  if (dtype >= 0) dtype &= ~(GATX_Q_UNPACKED | GATX_KV_UNPACKED);
  GATX_CALL(check_dims("diff_attention", dtype, heads, d, dv, E, std::max(rows, num_nodes)));
  if (rows == 0) return 0;
  GATX_REQUIRE(q && k && v && rowptr && col && lam && out, "diff_attention: null buffer");
  GATX_REQUIRE(nodes || rows == num_nodes, "diff_attention: a row for every node without nodes");
  GATX_REQUIRE(num_nodes > 0, "diff_attention: no nodes");
  GATX_REQUIRE(!plain_kv || (nodes && plain_q && d >= 8 && dv >= 8 && ldk >= 0 && ldv >= 0),
               "diff_attention: k and v as they come need nodes, q as it comes, d and dv >= 8");
  GATX_REQUIRE((plain_q ? ldq >= 0 : chunked(dtype, q, ldq)) &&
                   (plain_kv || (chunked(dtype, k, ldk) && chunked(dtype, v, ldv))),
               "diff_attention: rows of q, k, v must be 16-byte aligned (pack them)");
  GATX_REQUIRE(aligned16(out) && aligned16(order),
               "diff_attention: out and order must be 16-byte aligned");
  GATX_REQUIRE(!bias == !bucket, "diff_attention: bias and bucket go together");
  GATX_REQUIRE(nodes ? !S && !stat : S && stat,
               "diff_attention: S and stat hold whole rows' logits (not with nodes)");
  AttnArgs a = {};
  a.q = q; a.k = k; a.v = v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv;
  a.q_end = plain_q ? (rows - 1) * ldq + (int64_t)2 * heads * d : 0;
  a.kv_plain = plain_kv;
  a.d = d; a.dv = dv; a.dp = (int)round_up(d, 8); a.dvp = (int)round_up(dv, 8);
  a.col = col; a.E = E; a.scale = scale; a.lam = lam; a.bias = bias; a.bucket = bucket;
  a.S = (float2*)S; a.stat = (float4*)stat; a.out = out;
  a.part = (float*)part;
  const Geom g = attn_geom(d, dv);
  hipStream_t st = (hipStream_t)s;
  if (nodes) {
    GATX_REQUIRE(pieces >= 1 && pieces <= 4096, "diff_attention: 1..4096 pieces");
    const int64_t items = rows * heads * pieces;
    GATX_REQUIRE(items < (1ll << 31), "diff_attention: too many rows and pieces");
    GATX_REQUIRE(pieces == 1 || (part && part_bytes >= gatx_diff_attention_part_bytes(
                                             rows * pieces, heads, a.dvp)),
                 "diff_attention: workspace too small");
    a.part_width = 2 * a.dvp + 4;
    a.w.rows = (int)rows; a.w.num_nodes = num_nodes; a.w.heads = heads; a.w.rowptr = rowptr;
    a.w.nodes = nodes; a.w.pieces = pieces;
    a.w.gs = pieces > 1 ? 64 : row_lanes(g.G, items);
    a.w.gs_log = log2i(a.w.gs);
    const int64_t blocks = ceil_div(items, 256 / a.w.gs);
    const int64_t joins = pieces > 1 ? rows * heads * ceil_div(dv, kJoinCols) : 0;
    GATX_GRID(blocks, 256, "diff_attention");
    GATX_GRID(joins, 1024, "diff_attention");
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      with_geom(g, [&](auto G, auto NV) {
        constexpr int kG = decltype(G)::value, kNV = decltype(NV)::value;
        if (bias) diff_serve_kernel<T, kG, kNV, true><<<(unsigned)blocks, 256, 0, st>>>(a);
        else diff_serve_kernel<T, kG, kNV, false><<<(unsigned)blocks, 256, 0, st>>>(a);
      });
      return 0;
    });
    GATX_LAUNCH_CHECK("diff_attention_serve");
    if (pieces > 1) {
      with_dtype(dtype, [&](auto t) {
        diff_serve_join_kernel<decltype(t)><<<(unsigned)joins, 1024, 0, st>>>(a);
        return 0;
      });
      GATX_LAUNCH_CHECK("diff_attention_serve_join");
    }
    return 0;
  }
  GATX_REQUIRE(hub_edges == 0 || (hubs && hub_count), "diff_attention: null hub plan");
  const int64_t blocks = plan_rows(a.w, rows, heads, row_lanes(g.G, rows * heads), rowptr, order,
                                   hub_edges, hubs, hub_count, hub_bound);
  GATX_GRID(blocks, 256, "diff_attention");
  GATX_REQUIRE(a.w.hub_blocks == 0 ||
                   (part && part_bytes >= gatx_diff_attention_part_bytes(hub_bound, heads, a.dvp)),
               "diff_attention: workspace too small");
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    with_geom(Geom{g.G, 1}, [&](auto G, auto) {
      constexpr int kG = decltype(G)::value;
      if (bias) diff_score_kernel<T, kG, true><<<(unsigned)blocks, 256, 0, st>>>(a);
      else diff_score_kernel<T, kG, false><<<(unsigned)blocks, 256, 0, st>>>(a);
    });
    return 0;
  });
  GATX_LAUNCH_CHECK("diff_attention_score");
  if (a.w.hub_blocks) {
    diff_score_join_kernel<<<join_blocks(a.w, 256), 256, 0, st>>>(a);
    GATX_LAUNCH_CHECK("diff_attention_score_join");
  }
  a.part_width = a.dvp;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    with_geom(g, [&](auto G, auto NV) {
      diff_value_kernel<T, decltype(G)::value, decltype(NV)::value>
          <<<(unsigned)blocks, 256, 0, st>>>(a);
    });
    return 0;
  });
  GATX_LAUNCH_CHECK("diff_attention_value");
  if (a.w.hub_blocks) {
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      diff_sum_join_kernel<T><<<join_blocks(a.w, 1), 256, 0, st>>>(a, 0, nullptr, (T*)out);
      return 0;
    });
    GATX_LAUNCH_CHECK("diff_attention_value_join");
  }
  return 0;
}

namespace {
// Runs of slots of the bias gradient: enough waves to fill the chip, at least 1024 slots each.
int64_t bias_runs(int64_t E) { return std::max<int64_t>(1, std::min<int64_t>(512, E / 1024)); }
struct BackwardLayout {
  size_t dw, D, rec, lam, bias, part, total;
};
BackwardLayout backward_layout(int64_t N, int64_t E, int H, int dp, int dvp, int nb,
                               int64_t hub_bound, int64_t src_hub_bound) {
  BackwardLayout l = {};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t he = (size_t)H * E, hn = (size_t)H * N;
  l.rec = take(he * sizeof(float4));
  l.dw = take(he * sizeof(float));
  l.D = take(hn * sizeof(float2));
  l.lam = take(sizeof(double) * kLamRuns * H);
  l.bias = take(nb ? sizeof(float) * bias_runs(E) * H * nb : 0);
  l.part = take(sizeof(float) * std::max((size_t)hub_bound * H * (2 * dp),
                                         (size_t)src_hub_bound * H * (2 * dp + dvp)));
  l.total = at;
  return l;
}
}  // namespace

extern "C" size_t gatx_diff_attention_backward_workspace_bytes(int64_t N, int64_t E, int heads,
                                                               int d, int dv, int n_buckets,
                                                               int64_t hub_bound,
                                                               int64_t src_hub_bound) {
  return backward_layout(N, E, heads, (int)round_up(d, 8), (int)round_up(dv, 8), n_buckets,
                         hub_bound, src_hub_bound).total;
}

extern "C" int gatx_diff_attention_backward(
    int dtype, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
    const void* go, int64_t ldgo, int heads, int d, int dv, const int32_t* rowptr,
    const int32_t* col, const int32_t* srowptr, const int32_t* scol, const int32_t* seid, int64_t E,
    int64_t N, float scale, const float* lam, const uint8_t* bucket, int n_buckets, const float* S,
    const float* stat, void* gq, void* gk, void* gv, float* glam, float* gbias, int hub_edges,
    const int32_t* hubs, const int32_t* hub_count, int64_t hub_bound, const int32_t* src_hubs,
    const int32_t* src_hub_count, int64_t src_hub_bound, void* workspace, size_t workspace_bytes,
    const int32_t* order, const int32_t* src_order, gatx_stream_t s) {
  GATX_CALL(check_dims("diff_attention_backward", dtype, heads, d, dv, E, N));
  GATX_REQUIRE(n_buckets >= 0 && n_buckets <= kMaxBuckets, "diff_attention_backward: %d buckets",
               n_buckets);
  GATX_REQUIRE(!gbias || (bucket && n_buckets > 0), "diff_attention_backward: null bucket");
  hipStream_t st = (hipStream_t)s;
  if (N == 0) {
    if (glam) zero_words_kernel<<<(unsigned)ceil_div(heads, 64), 64, 0, st>>>((uint32_t*)glam, heads);
    if (gbias)
      zero_words_kernel<<<(unsigned)ceil_div(n_buckets * heads, 64), 64, 0, st>>>(
          (uint32_t*)gbias, n_buckets * heads);
    GATX_LAUNCH_CHECK("diff_attention_backward zero");
    return 0;
  }
  const bool by_source = gk || gv;
  GATX_REQUIRE(aligned16(gq) && aligned16(gk) && aligned16(gv) && aligned16(order) &&
                   aligned16(src_order),
               "diff_attention_backward: gradients and orders must be 16-byte aligned");
  GATX_REQUIRE(q && k && v && go && rowptr && col && lam && S && stat,
               "diff_attention_backward: null buffer");
  GATX_REQUIRE(!by_source || (srowptr && scol && seid), "diff_attention_backward: null transpose");
  GATX_REQUIRE(chunked(dtype, q, ldq) && chunked(dtype, k, ldk) && chunked(dtype, v, ldv) &&
               chunked(dtype, go, ldgo),
               "diff_attention_backward: rows of q, k, v, go must be 16-byte aligned (pack them)");
  // each direction with its plan or without (NULL: it has no long rows, or walks them whole)
  GATX_REQUIRE(hub_edges >= 0 && hub_bound >= 0 && src_hub_bound >= 0 && !hubs == !hub_count &&
                   !src_hubs == !src_hub_count && (hubs || hub_bound == 0) &&
                   (src_hubs || src_hub_bound == 0) && (hub_edges == 0 || hubs || src_hubs),
               "diff_attention_backward: bad hub plan");
  const int dp = (int)round_up(d, 8), dvp = (int)round_up(dv, 8);
  const BackwardLayout l =
      backward_layout(N, E, heads, dp, dvp, gbias ? n_buckets : 0, hub_bound, src_hub_bound);
  GATX_REQUIRE(workspace && workspace_bytes >= l.total,
               "diff_attention_backward: workspace too small");
  char* ws = (char*)workspace;
  AttnArgs a = {};
  a.q = q; a.k = k; a.v = v; a.go = go; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldgo = ldgo;
  a.d = d; a.dv = dv; a.dp = dp; a.dvp = dvp; a.col = col; a.E = E; a.scale = scale; a.lam = lam;
  a.S = (float2*)const_cast<float*>(S); a.stat = (float4*)const_cast<float*>(stat);
  a.dw = (float*)(ws + l.dw); a.D = (float2*)(ws + l.D); a.rec = (float4*)(ws + l.rec);
  a.part = (float*)(ws + l.part);
  a.gq = gq; a.gk = gk; a.gv = gv;
  const Geom g = attn_geom(d, dv);
  const int gs = row_lanes(g.G, N * heads);
  // A
  int64_t blocks = plan_rows(a.w, N, heads, gs, rowptr, order, hub_edges, hubs, hub_count,
                             hub_bound);
  GATX_GRID(blocks, 256, "diff_attention_backward");
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    with_geom(g, [&](auto G, auto NV) {
      diff_dw_kernel<T, decltype(G)::value, decltype(NV)::value>
          <<<(unsigned)blocks, 256, 0, st>>>(a);
    });
    return 0;
  });
  GATX_LAUNCH_CHECK("diff_attention_dw");
  if (a.w.hub_blocks) {
    diff_dw_join_kernel<<<join_blocks(a.w, 256), 256, 0, st>>>(a);
    GATX_LAUNCH_CHECK("diff_attention_dw_join");
  }
  if (glam) {
    const int runs = (int)std::min<int64_t>(kLamRuns, ceil_div(N, 1024));
    double* lp = (double*)(ws + l.lam);
    diff_lam_kernel<<<dim3(runs, heads), 256, 0, st>>>(a.D, N, ceil_div(N, runs), lp, glam);
    GATX_LAUNCH_CHECK("diff_attention_lam");
    if (runs > 1) {
      diff_lam_join_kernel<<<(unsigned)ceil_div(heads, 64), 64, 0, st>>>(lp, runs, heads, glam);
      GATX_LAUNCH_CHECK("diff_attention_lam_join");
    }
  }
  // B
  if (gq || by_source || gbias) {
    a.part_width = 2 * dp;
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      with_geom(Geom{g.G, 1}, [&](auto G, auto) {
        diff_gq_kernel<T, decltype(G)::value><<<(unsigned)blocks, 256, 0, st>>>(a);
      });
      return 0;
    });
    GATX_LAUNCH_CHECK("diff_attention_gq");
    if (a.w.hub_blocks && gq) {
      with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        diff_sum_join_kernel<T><<<join_blocks(a.w, 1), 256, 0, st>>>(a, 1, (T*)gq, nullptr);
        return 0;
      });
      GATX_LAUNCH_CHECK("diff_attention_gq_join");
    }
  }
  if (gbias) {
    const int64_t runs = bias_runs(E);
    float* bp = (float*)(ws + l.bias);
    diff_bias_kernel<<<dim3((unsigned)runs, heads), 64, sizeof(float) * 64 * n_buckets, st>>>(
        a.rec, bucket, rowptr, N, E, ceil_div(E, runs), n_buckets, bp);
    GATX_LAUNCH_CHECK("diff_attention_bias");
    diff_bias_join_kernel<<<dim3(n_buckets, heads), 64, 0, st>>>(bp, (int)runs, n_buckets, heads,
                                                                 gbias);
    GATX_LAUNCH_CHECK("diff_attention_bias_join");
  }
  // C
  if (by_source) {
    a.col = scol;
    a.seid = seid;
    a.part_width = 2 * dp + dvp;
    blocks = plan_rows(a.w, N, heads, gs, srowptr, src_order, hub_edges, src_hubs,
                       src_hub_count, src_hub_bound);
    GATX_GRID(blocks, 256, "diff_attention_backward");
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      with_geom(g, [&](auto G, auto NV) {
        diff_gkv_kernel<T, decltype(G)::value, decltype(NV)::value>
            <<<(unsigned)blocks, 256, 0, st>>>(a);
      });
      return 0;
    });
    GATX_LAUNCH_CHECK("diff_attention_gkv");
    if (a.w.hub_blocks) {
      with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        diff_sum_join_kernel<T><<<join_blocks(a.w, 1), 256, 0, st>>>(a, 1, (T*)gk, (T*)gv);
        return 0;
      });
      GATX_LAUNCH_CHECK("diff_attention_gkv_join");
    }
  }
  return 0;
}
