// The norms around a block, with its gate and residual scale, in one pass over the rows:
//   y    = resid + scale * sigmoid(gate) * weight * h rh,   rh = 1 / sqrt(mean h^2 + eps)
//   next = next_weight * y ry,                              ry = 1 / sqrt(mean y^2 + eps)
// and its gradients. With hn = h rh, yn = y ry, c = scale sigmoid(gate) weight:
//   u   = gn next_weight;   g = gy + ry (u - yn mean(u yn))         (the gradient of y)
//   gresid = g;  t = g c;   gh = rh (t - hn mean(t hn))
//   ggate = g c hn sigmoid(-gate)                    (1 - sigmoid(gate) would cancel where a gate is open)
// The parameters' gradients are column sums of two products only: A = sum g sigmoid(gate) hn and
// B = sum gn yn give gweight = scale A, gscale = weight A, gnext = B and, for a gate that is a
// parameter, ggate = scale weight sigmoid(-gate) A.
//
// HBM-bound: every input is read once and every output written once, a row's values stay in
// registers between the two norms (y is not rounded on the way to the second one). One group of
// lanes per row: 8..64 lanes of a wave up to 128 16-byte chunks a row, else a whole workgroup, so a
// lane holds at most 16 elements of each stream (the backward has five of them and two sums). The
// backward's workgroups walk the rows in a fixed stride and keep A and B in registers; their
// partial sums are added in workgroup order by a second launch.
//
// 44 900 x 1024 bf16, every part there: forward 82 us (460 MB, 5.6 TB/s), backward 199 (736 MB, 3.7
// TB/s: the loads of a row wait for its two sums), column sums 5.
//
// Rows that are no whole 16-byte chunks (by their width, stride or address) are read and written
// element by element, which costs 1.5 to 4 times as much: 44 900 x 726 bf16 317 + 474 us (728
// columns: 73 + 186), 8192 x 1997 bf16 83 + 203 (2000: 27 + 82), float32 126 + 255 (59 + 115).
#include "dtypes.h"

namespace gatx {
namespace {

constexpr int kMaxCols = 8192;
// Workgroups of the backward (their column partials): 3 a CU are what the registers of 16 elements of
// five streams leave. 44 900 x 1024 bf16, before both_parts: 194 us with 768, 254 with 512, 255 with
// 1024 (a second round for a quarter of them), 200 with 1536; 128 registers (4 a CU) spill: 344 us; the next row's
// loads in flight as well, or keeping a row unwidened between its two sums, cost the waves they need:
// 262 and 277 us. A copy of the same bytes takes 144 us.
constexpr int kMaxParts = 768;

struct NormArgs {
  const void *h, *resid, *gate, *gy, *gn;
  int64_t ldh, ldr, ldg, ldgy, ldgn;
  const float *weight, *scale, *next_weight;
  const float *rstd_h, *rstd_y;          // backward
  float *rstd_h_out, *rstd_y_out;        // forward
  void *y, *next, *gh, *gresid, *ggate;  // packed
  float* part;                           // [parts][2][cols]
  int64_t rows;
  int cols, gate_rows, lanes;
  float eps;
};

__device__ inline float lanes_sum(float v, int lanes) {
  switch (lanes) {
    case 8: return group_sum<8>(v);
    case 16: return group_sum<16>(v);
    case 32: return group_sum<32>(v);
    default: return group_sum<64>(v);
  }
}

// Sum over the lanes that share a row, in every one of them. BLOCK: the whole workgroup, through
// LDS (the barrier before the write keeps one row's readers ahead of the next row's writers).
template <bool BLOCK>
__device__ inline float row_sum(float v, int lanes, float* red) {
  if (!BLOCK) return lanes_sum(v, lanes);
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
  return s;
}

template <int N>
__device__ inline void fill(float (&v)[N], float x) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = x;
}

// BLOCK: the workgroup's lanes share a row, else `lanes` of a wave do. Lane li of the row holds the
// chunks li, li + lanes, ... (CH of them, VEC elements each).
template <typename T, int VEC, int CH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) norm_forward_kernel(NormArgs a) {
  __shared__ float red[16];
  const int lanes = BLOCK ? (int)blockDim.x : a.lanes;
  const int li = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1));
  const int64_t r = BLOCK ? (int64_t)blockIdx.x
                          : (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const bool live = r < a.rows;
  const int64_t rr = live ? r : 0;   // spare groups of the last workgroup read row 0
  const float inv_n = 1.f / (float)a.cols;
  float y[CH][VEC];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * lanes + li) * VEC;
    fill(y[c], 0.f);
    if (col < a.cols) load_f32((const T*)a.h + rr * a.ldh + col, y[c]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss = fmaf(y[c][i], y[c][i], ss);
  }
  if (a.weight) {
    const float rh = rsqrtf(row_sum<BLOCK>(ss, lanes, red) * inv_n + a.eps);
    if (live && li == 0 && a.rstd_h_out) a.rstd_h_out[r] = rh;
    ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * lanes + li) * VEC;
      if (col >= a.cols) continue;
      float w[VEC], x[VEC];
      load_f32(a.weight + col, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[c][i] *= rh * w[i];
      if (a.scale) {
        load_f32(a.scale + col, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] *= x[i];
      }
      if (a.gate) {
        if (a.gate_rows) load_f32((const T*)a.gate + rr * a.ldg + col, x);
        else load_f32((const float*)a.gate + col, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] *= sigmoid(x[i]);
      }
      if (a.resid) {
        load_f32((const T*)a.resid + rr * a.ldr + col, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] += x[i];
      }
      if (live && a.y) store_f32((T*)a.y + r * a.cols + col, y[c]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(y[c][i], y[c][i], ss);
    }
  }
  if (!a.next) return;
  const float ry = rsqrtf(row_sum<BLOCK>(ss, lanes, red) * inv_n + a.eps);
  if (!live) return;
  if (li == 0 && a.rstd_y_out) a.rstd_y_out[r] = ry;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * lanes + li) * VEC;
    if (col >= a.cols) continue;
    float w[VEC];
    load_f32(a.next_weight + col, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] *= y[c][i] * ry;
    store_f32((T*)a.next + r * a.cols + col, w);
  }
}

// sigmoid(gate) and sigmoid(-gate) in one number: the smaller of them, whose difference from 1 is the
// other to its last bit, with the sign set where that is sigmoid(-gate). The gradient of a gate needs
// both, and 1 - sigmoid(gate) is nothing but rounding where a gate is open. (44 900 x 1024 bf16: 199
// us; 195 with that difference; 212 with the gate loaded again for sigmoid(-gate).)
__device__ inline float both_parts(float gate) {
  const float t = __expf(-fabsf(gate));
  return copysignf(t / (1.f + t), -gate);
}
__device__ inline bool is_open(float s) { return __float_as_int(s) < 0; }
__device__ inline float open_part(float s) { return s + (is_open(s) ? 1.f : 0.f); }
__device__ inline float shut_part(float s) { return (is_open(s) ? 0.f : 1.f) - s; }

template <typename T, int VEC, int CH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) norm_backward_kernel(NormArgs a) {
  __shared__ float red[16];
  extern __shared__ __attribute__((aligned(16))) float sums[];   // group form: [groups][2][cols]
  const int lanes = BLOCK ? (int)blockDim.x : a.lanes;
  const int li = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1));
  const int groups = BLOCK ? 1 : 256 / lanes;
  const int grp = BLOCK ? 0 : (int)threadIdx.x / lanes;
  const float inv_n = 1.f / (float)a.cols;
  float A[CH][VEC], B[CH][VEC];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    fill(A[c], 0.f);
    fill(B[c], 0.f);
  }
  // every lane of the workgroup makes the same number of turns (the row sums need all of them)
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += (int64_t)gridDim.x * groups) {
    const int64_t r = r0 + grp;
    const bool live = r < a.rows;
    const int64_t rr = live ? r : 0;
    // hn, the gate's factors and y; g starts as gy
    float hn[CH][VEC], sg[CH][VEC], y[CH][VEC], g[CH][VEC], gn[CH][VEC];
    const float rh = a.weight ? a.rstd_h[rr] : 1.f;
    const float ry = a.gn ? a.rstd_y[rr] : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * lanes + li) * VEC;
      fill(hn[c], 0.f);
      fill(sg[c], -0.f);   // no gate: open
      fill(g[c], 0.f);
      fill(gn[c], 0.f);
      fill(y[c], 0.f);
      if (col >= a.cols) continue;
      load_f32((const T*)a.h + rr * a.ldh + col, hn[c]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) hn[c][i] *= rh;
      if (a.gate) {
        if (a.gate_rows) load_f32((const T*)a.gate + rr * a.ldg + col, sg[c]);
        else load_f32((const float*)a.gate + col, sg[c]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sg[c][i] = both_parts(sg[c][i]);
      }
      if (a.gy) load_f32((const T*)a.gy + rr * a.ldgy + col, g[c]);
      if (a.gn) {
        float w[VEC], x[VEC];
        load_f32((const T*)a.gn + rr * a.ldgn + col, gn[c]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] = hn[c][i];
        if (a.weight) {
          load_f32(a.weight + col, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[c][i] *= w[i] * open_part(sg[c][i]);
          if (a.scale) {
            load_f32(a.scale + col, w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) y[c][i] *= w[i];
          }
          if (a.resid) {
            load_f32((const T*)a.resid + rr * a.ldr + col, x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) y[c][i] += x[i];
          }
        }
        load_f32(a.next_weight + col, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y[c][i] *= ry;   // yn
          if (live) B[c][i] = fmaf(gn[c][i], y[c][i], B[c][i]);
          gn[c][i] *= w[i];   // u
          dot = fmaf(gn[c][i], y[c][i], dot);
        }
      }
    }
    if (a.gn) {
      const float m = row_sum<BLOCK>(dot, lanes, red) * inv_n;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[c][i] += ry * (gn[c][i] - y[c][i] * m);
    }
    if (!a.weight) {   // y = h: the norm before a block alone
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (c * lanes + li) * VEC;
        if (live && col < a.cols && a.gh) store_f32((T*)a.gh + r * a.cols + col, g[c]);
      }
      continue;
    }
    dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * lanes + li) * VEC;
      if (col >= a.cols) continue;
      float w[VEC], x[VEC];
      if (live && a.gresid) store_f32((T*)a.gresid + r * a.cols + col, g[c]);
      load_f32(a.weight + col, w);
      if (a.scale) {
        load_f32(a.scale + col, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] *= x[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float gs = g[c][i] * open_part(sg[c][i]);
        if (live) A[c][i] = fmaf(gs, hn[c][i], A[c][i]);
        g[c][i] = gs * w[i];   // t
        x[i] = g[c][i] * hn[c][i];
        dot += x[i];
        x[i] *= shut_part(sg[c][i]);
      }
      if (live && a.ggate && a.gate_rows) store_f32((T*)a.ggate + r * a.cols + col, x);
    }
    const float m = row_sum<BLOCK>(dot, lanes, red) * inv_n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * lanes + li) * VEC;
      if (!live || col >= a.cols || !a.gh) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[c][i] = rh * (g[c][i] - hn[c][i] * m);
      store_f32((T*)a.gh + r * a.cols + col, g[c]);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
  if (BLOCK) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * lanes + li) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col < a.cols) {
          part[col + i] = A[c][i];
          part[a.cols + col + i] = B[c][i];
        }
    }
    return;
  }
  float* mine = sums + (int64_t)grp * 2 * a.cols;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * lanes + li) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (col < a.cols) {
        mine[col + i] = A[c][i];
        mine[a.cols + col + i] = B[c][i];
      }
  }
  __syncthreads();
  for (int col = threadIdx.x; col < 2 * a.cols; col += 256) {
    float s = 0.f;
    for (int k = 0; k < groups; ++k) s += sums[(int64_t)k * 2 * a.cols + col];
    part[col] = s;
  }
}

// The workgroups' partial sums added in order, 32 columns a workgroup, and the parameters'
// gradients from them. blockIdx.y: A (0) or B (1).
__global__ void __launch_bounds__(1024) norm_columns_kernel(NormArgs a, int parts, float* gweight,
                                                            float* gscale, float* gnext) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, gy = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + cx;
  if (blockIdx.y == 0 && !a.weight) return;   // the norm before a block has no A
  float s = 0.f;
  if (col < a.cols) {
    const float* p = a.part + (int64_t)blockIdx.y * a.cols + col;
#pragma unroll 8
    for (int k = gy; k < parts; k += 32) s += p[(int64_t)k * 2 * a.cols];
  }
  red[gy][cx] = s;
  __syncthreads();
  if (gy != 0 || col >= a.cols) return;
  s = 0.f;
  for (int k = 0; k < 32; ++k) s += red[k][cx];
  if (blockIdx.y == 1) {
    if (gnext) gnext[col] = s;
    return;
  }
  const float w = a.weight[col], sc = a.scale ? a.scale[col] : 1.f;
  if (gweight) gweight[col] = sc * s;
  if (gscale) gscale[col] = w * s;
  if (a.ggate && !a.gate_rows)
    ((float*)a.ggate)[col] = sc * w * sigmoid(-((const float*)a.gate)[col]) * s;
}

// How a row is dealt out: `lanes` lanes with `ch` chunks each; lanes > 64: a workgroup.
struct NormGeom {
  int vec, lanes, ch;
  bool block() const { return lanes > 64; }
  int rows_per_block() const { return block() ? 1 : 256 / lanes; }
};
NormGeom norm_geom(int dtype, int64_t cols, bool aligned) {
  const int vec = aligned ? 16 / dtype_size(dtype) : 1;
  const int n = (int)ceil_div(cols, vec);
  if (n <= 64) {
    int l = 8;
    while (l < n) l <<= 1;
    return {vec, l, 1};
  }
  if (n <= 128) return {vec, 64, 2};
  if (n <= 512) return {vec, n <= 256 ? 256 : 512, 1};
  int ch = 1;
  while (ch * 1024 < n) ch <<= 1;
  return {vec, 1024, ch};
}

template <typename T, int VEC, int CH, bool BLOCK>
void launch(const NormArgs& a, const NormGeom& g, bool backward, int64_t blocks, hipStream_t st) {
  const int threads = BLOCK ? g.lanes : 256;
  if (!backward) {
    norm_forward_kernel<T, VEC, CH, BLOCK><<<(unsigned)blocks, threads, 0, st>>>(a);
  } else {
    const size_t lds = BLOCK || !a.part ? 0 : sizeof(float) * 2 * a.cols * (256 / g.lanes);
    norm_backward_kernel<T, VEC, CH, BLOCK><<<(unsigned)blocks, threads, lds, st>>>(a);
  }
}

template <typename T, int VEC>
void dispatch(const NormArgs& a, const NormGeom& g, bool backward, int64_t blocks, hipStream_t st) {
  if (!g.block()) {
    if (g.ch == 1) launch<T, VEC, 1, false>(a, g, backward, blocks, st);
    else launch<T, VEC, 2, false>(a, g, backward, blocks, st);
  } else if (g.ch == 1) {
    launch<T, VEC, 1, true>(a, g, backward, blocks, st);
  } else if constexpr (VEC < 8) {   // 8192 columns: at most 1 chunk of 8, 2 of 4, 8 of 1
    if (g.ch == 2) launch<T, VEC, 2, true>(a, g, backward, blocks, st);
    else if constexpr (VEC == 1) {
      if (g.ch == 4) launch<T, VEC, 4, true>(a, g, backward, blocks, st);
      else launch<T, VEC, 8, true>(a, g, backward, blocks, st);
    }
  }
}

int run_norm(int dtype, const NormArgs& a, const NormGeom& g, bool backward, int64_t blocks,
             hipStream_t st) {
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (g.vec == 1) dispatch<T, 1>(a, g, backward, blocks, st);
    else dispatch<T, 16 / sizeof(T)>(a, g, backward, blocks, st);
    return 0;
  });
}

// Whole 16-byte chunks in every row of every stream, and in the parameters.
bool rows_aligned(int dtype, int64_t cols, std::initializer_list<std::pair<const void*, int64_t>> s,
                  std::initializer_list<const void*> packed) {
  const int vec = 16 / dtype_size(dtype);
  if (cols % vec) return false;
  for (auto& x : s)
    if (x.first && (!aligned16(x.first) || x.second % vec)) return false;
  for (auto* p : packed)
    if (p && !aligned16(p)) return false;
  return true;
}

int64_t norm_parts(int64_t rows, const NormGeom& g) {
  return std::min<int64_t>(ceil_div(rows, g.rows_per_block()), kMaxParts);
}

}  // namespace
}  // namespace gatx

using namespace gatx;

extern "C" int gatx_block_norm(int dtype, int64_t rows, int64_t cols, const void* h, int64_t ldh,
                               const float* weight, const void* resid, int64_t ldr,
                               const void* gate, int gate_rows, int64_t ldg, const float* scale,
                               const float* next_weight, float eps, void* y, void* next,
                               float* rstd_h, float* rstd_y, gatx_stream_t s) {
  GATX_REQUIRE(dtype_ok(dtype), "block_norm: unknown dtype %d", dtype);
  GATX_REQUIRE(rows >= 0 && cols >= 1 && cols <= kMaxCols, "block_norm: %lld columns (1..%d)",
               (long long)cols, kMaxCols);
  if (rows == 0) return 0;
  GATX_REQUIRE(weight || (!resid && !gate && !scale && !y), "block_norm: weight missing");
  GATX_REQUIRE(h, "block_norm: null input");
  GATX_REQUIRE(weight || next, "block_norm: no output");
  GATX_REQUIRE(!next == !next_weight, "block_norm: next and next_weight go together");
  NormArgs a = {};
  a.h = h; a.ldh = ldh; a.weight = weight; a.resid = resid; a.ldr = ldr; a.gate = gate;
  a.gate_rows = gate_rows; a.ldg = ldg; a.scale = scale; a.next_weight = next_weight; a.eps = eps;
  a.y = y; a.next = next; a.rstd_h_out = rstd_h; a.rstd_y_out = rstd_y;
  a.rows = rows; a.cols = (int)cols;
  const NormGeom g = norm_geom(dtype, cols, rows_aligned(
      dtype, cols, {{h, ldh}, {resid, ldr}, {gate_rows ? gate : nullptr, ldg}},
      {gate, weight, scale, next_weight, y, next}));
  a.lanes = g.lanes;
  const int64_t blocks = ceil_div(rows, g.rows_per_block());
  // a launch holds fewer than 2^32 threads (taking turns in a loop costs every call 4%)
  GATX_REQUIRE(blocks * (g.block() ? g.lanes : 256) < (1ll << 32), "block_norm: too many rows");
  run_norm(dtype, a, g, false, blocks, (hipStream_t)s);
  GATX_LAUNCH_CHECK("block_norm");
  return 0;
}

extern "C" size_t gatx_block_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  return sizeof(float) * 2 * (size_t)std::min<int64_t>(rows, kMaxParts) * (size_t)cols;
}

extern "C" int gatx_block_norm_backward(int dtype, int64_t rows, int64_t cols, const void* h,
                                        int64_t ldh, const float* weight, const void* resid,
                                        int64_t ldr, const void* gate, int gate_rows, int64_t ldg,
                                        const float* scale, const float* next_weight,
                                        const float* rstd_h, const float* rstd_y, const void* gy,
                                        int64_t ldgy, const void* gn, int64_t ldgn, void* gh,
                                        void* gresid, void* ggate, float* gweight, float* gscale,
                                        float* gnext, void* workspace, size_t workspace_bytes,
                                        gatx_stream_t s) {
  GATX_REQUIRE(dtype_ok(dtype), "block_norm_backward: unknown dtype %d", dtype);
  GATX_REQUIRE(rows >= 0 && cols >= 1 && cols <= kMaxCols,
               "block_norm_backward: %lld columns (1..%d)", (long long)cols, kMaxCols);
  const bool params = gweight || gscale || gnext || (ggate && !gate_rows);
  if (rows == 0) {   // empty sums (a kernel's fill: the call may be captured)
    float* const outs[] = {gweight, gscale, gnext, gate_rows ? nullptr : (float*)ggate};
    for (float* p : outs)
      if (p) zero_words_kernel<<<(unsigned)ceil_div(cols, 256), 256, 0, (hipStream_t)s>>>(
          (uint32_t*)p, cols);
    GATX_LAUNCH_CHECK("block_norm_backward zero");
    return 0;
  }
  GATX_REQUIRE(weight || (!resid && !gate && !scale && !gresid && !ggate && !gweight && !gscale),
               "block_norm_backward: weight missing");
  GATX_REQUIRE(!gn || next_weight, "block_norm_backward: next_weight missing");
  GATX_REQUIRE(h && (!weight || rstd_h) && (!gn || rstd_y), "block_norm_backward: null input");
  GATX_REQUIRE(!params || (workspace && workspace_bytes >=
                           gatx_block_norm_backward_workspace_bytes(rows, cols)),
               "block_norm_backward: workspace too small");
  NormArgs a = {};
  a.h = h; a.ldh = ldh; a.weight = weight; a.resid = resid; a.ldr = ldr; a.gate = gate;
  a.gate_rows = gate_rows; a.ldg = ldg; a.scale = scale; a.next_weight = next_weight;
  a.rstd_h = rstd_h; a.rstd_y = rstd_y; a.gy = gy; a.ldgy = ldgy; a.gn = gn; a.ldgn = ldgn;
  a.gh = gh; a.gresid = gresid; a.ggate = ggate;
  a.rows = rows; a.cols = (int)cols;
  a.part = params ? (float*)workspace : nullptr;
  const NormGeom g = norm_geom(dtype, cols, rows_aligned(
      dtype, cols, {{h, ldh}, {resid, ldr}, {gate_rows ? gate : nullptr, ldg}, {gy, ldgy},
                    {gn, ldgn}},
      {gate, weight, scale, next_weight, gh, gresid, ggate}));
  a.lanes = g.lanes;
  const int64_t parts = norm_parts(rows, g);
  run_norm(dtype, a, g, true, parts, (hipStream_t)s);
  GATX_LAUNCH_CHECK("block_norm_backward");
  if (params) {
    const dim3 grid((unsigned)ceil_div(cols, 32), gnext ? 2 : 1);
    norm_columns_kernel<<<grid, 1024, 0, (hipStream_t)s>>>(a, (int)parts, gweight, gscale, gnext);
    GATX_LAUNCH_CHECK("block_norm_columns");
  }
  return 0;
}
