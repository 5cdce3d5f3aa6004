// Distillation from a teacher's top logits: loss_i = T^2 sum_k p_k (log p_k - log q[c_k]) with
// p = softmax over the row's K kept teacher logits of t / T and q = softmax over all classes of
// s / T; d loss_i / d s_j = T (q_j - sum of the p_k with c_k = j).
//
// HBM-bound: the forward streams the logits once (a running maximum and sum a lane, joined at the
// end), the backward streams them again and writes the gradient, from the two maxima and sums that
// the forward kept (16 bytes a row) rather than a stored gradient of the size of the logits, which
// would have to be scaled, and so read and written, once more. The gradient is written as g T q
// first; the row's few taught classes are then written again by the same workgroup, the slots of
// one class added in slot order, so the result does not depend on the order of anything.
//
// 8192 x 32000 bf16, K = 64: forward 149 us (3.5 TB/s; a plain read of the logits 140), backward 200
// (5.2 TB/s; their copy 205). 44 900 x 121 float32, K = 16: 20 + 22 us (1.5 and 2.4 TB/s, of logits
// that the L2s and the memory-side cache hold): far from the bytes (10 us for both) and from the exp2
// (one a logit). What is left is each row's chain of dependent exchanges between its lanes, some 25 of
// them in the forward (a maximum and sum, two maxima, two sums, log2(lanes) steps each); not timed apart.
//
// Taught classes cost K^2 LDS reads a row in the backward (each slot looks for others of its class):
// nothing at K = 64, but 8192 x 32000 bf16 takes 307 us at K = 256 and 2630 at the most slots, 1024.
//
// Rows of up to 1024 classes and 64 slots: a group of 8..64 lanes of a wave each, walking the rows
// in a fixed stride. Wider rows: a workgroup each, 16-byte accesses from the first aligned element
// on (rows of an odd number of classes start anywhere).
#include "dtypes.h"

namespace gatx {
namespace {

constexpr int kMaxSlots = 1024;
constexpr int kGroupSlots = 64, kGroupClasses = 1024;
constexpr int kMaxBlocks = 8192;
constexpr int kFlight = 4;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_huge_valf();

struct DistillArgs {
  const void *logits, *teacher, *index;
  int64_t rows, ld;
  int classes, K, teacher_dtype, index64, lanes;
  float T, k;        // k = log2(e) / T
  float* row_loss;
  float* part;       // [blocks][2]: loss, rows with slots
  float* stat;       // [rows][4]: max s, log2 sum, max t, log2 sum (the last -inf: no slots)
  const float *g, *count;
  int g_stride;
  void* grad;
};

__device__ inline float teacher_at(const DistillArgs& a, int64_t i) {
  if (a.teacher_dtype == GATX_F32) return ((const float*)a.teacher)[i];
  if (a.teacher_dtype == GATX_BF16) return (float)((const __bf16*)a.teacher)[i];
  return (float)((const _Float16*)a.teacher)[i];
}
// The slot's class; -1: empty. Classes past the last one stay what they are (as INT_MAX).
__device__ inline int class_at(const DistillArgs& a, int64_t i) {
  const int64_t c = a.index64 ? ((const int64_t*)a.index)[i] : ((const int32_t*)a.index)[i];
  return c < 0 ? -1 : c >= a.classes ? 0x7fffffff : (int)c;
}

// Running maximum and sum of exp2((x - m) k).
struct Lse {
  float m = -kInf, s = 0.f;
};
template <int N>
__device__ inline void lse_add(Lse& z, const float (&x)[N], float k) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, x[i]);
  mx = fmaxf(mx, z.m);
  const float ref = mx == -kInf ? 0.f : mx;   // nothing but -inf so far: every term is 0
  float s = z.s * __builtin_amdgcn_exp2f((z.m - ref) * k);
#pragma unroll
  for (int i = 0; i < N; ++i) s += __builtin_amdgcn_exp2f((x[i] - ref) * k);
  z.m = mx;
  z.s = s;
}
__device__ inline void lse_join(Lse& z, float m, float s, float k) {
  const float mx = fmaxf(z.m, m), ref = mx == -kInf ? 0.f : mx;
  z.s = z.s * __builtin_amdgcn_exp2f((z.m - ref) * k) + s * __builtin_amdgcn_exp2f((m - ref) * k);
  z.m = mx;
}
__device__ inline void lse_join_lanes(Lse& z, int lanes, float k) {
  for (int d = 1; d < lanes; d <<= 1) {
    const float m = __shfl_xor(z.m, d), s = __shfl_xor(z.s, d);
    // both partners add the same two terms in the same order
    const bool low = !(threadIdx.x & d);
    Lse lo{low ? z.m : m, low ? z.s : s};
    lse_join(lo, low ? m : z.m, low ? s : z.s, k);
    z = lo;
  }
}
__device__ inline float lanes_total(float v, int lanes) {
  for (int d = 1; d < lanes; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ inline float lanes_most(float v, int lanes) {
  for (int d = 1; d < lanes; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// A slot: its class (-1: empty) and teacher logit. Both loads are issued at once and used later, so a
// lane's first slot is on its way while the row's logits are.
struct Slot {
  int c = -1;
  float t = -kInf;
  __device__ Slot(const DistillArgs& a, int64_t at, int j) {
    const int k = min(j, a.K - 1);
    const int cls = class_at(a, at + k);
    const float x = teacher_at(a, at + k);
    if (j < a.K && cls >= 0 && x != -kInf) {
      c = cls;
      t = x;
    }
  }
  __device__ bool there() const { return c >= 0; }
  __device__ bool past() const { return c == 0x7fffffff; }
};
// f(slot) for a lane's slots li, li + lanes, ... that are not empty; `first` is slot li.
template <typename F>
__device__ inline void each_slot(const DistillArgs& a, const Slot& first, int64_t at, int li,
                                 int lanes, F&& f) {
  if (first.there()) f(first);
  for (int j = li + lanes; j < a.K; j += lanes) {
    const Slot s(a, at, j);
    if (s.there()) f(s);
  }
}
// One row's teacher: a lane's largest logit, and whether a slot is out of range or NaN.
__device__ inline float teacher_max(const DistillArgs& a, const Slot& first, int64_t at, int li,
                                    int lanes, bool& bad) {
  float tm = -kInf;
  bad = false;
  each_slot(a, first, at, li, lanes, [&](const Slot& s) {
    bad |= s.past() || s.t != s.t;
    tm = fmaxf(tm, s.t);
  });
  return tm;
}
__device__ inline float teacher_sum(const DistillArgs& a, const Slot& first, int64_t at, int li,
                                    int lanes, float tm) {
  float ts = 0.f;
  each_slot(a, first, at, li, lanes,
            [&](const Slot& s) { ts += __builtin_amdgcn_exp2f((s.t - tm) * a.k); });
  return ts;
}
// Its share of sum_k p_k (log p_k - log q[c_k]), in units of ln 2: the logarithms are base 2.
template <typename T>
__device__ inline float slots_loss(const DistillArgs& a, const T* row, const Slot& first,
                                   int64_t at, int li, int lanes, float m, float ls, float tm,
                                   float lts) {
  float sum = 0.f;
  each_slot(a, first, at, li, lanes, [&](const Slot& s) {
    if (s.past()) return;
    const float lp = (s.t - tm) * a.k - lts, p = __builtin_amdgcn_exp2f(lp);
    if (p > 0.f) sum += p * (lp - (((float)row[s.c] - m) * a.k - ls));
    else if (p != p) sum = p;
  });
  return sum;
}

template <typename T>
__global__ void __launch_bounds__(256) distill_group_kernel(DistillArgs a) {
  __shared__ float red[2][32];
  const int lanes = a.lanes, li = threadIdx.x & (lanes - 1), grp = threadIdx.x / lanes;
  const int groups = 256 / lanes;
  float total = 0.f, some = 0.f;
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += (int64_t)gridDim.x * groups) {
    const int64_t r = r0 + grp;
    if (r >= a.rows) continue;   // whole groups drop out; exchanges stay within a group
    const T* row = (const T*)a.logits + r * a.ld;
    const int64_t at = r * a.K;
    const Slot slot(a, at, li);
    Lse z;
    for (int c = li; c < a.classes; c += 4 * lanes) {
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = (float)row[min(c + u * lanes, a.classes - 1)];
#pragma unroll
      for (int u = 1; u < 4; ++u) x[u] = c + u * lanes < a.classes ? x[u] : -kInf;
      lse_add(z, x, a.k);
    }
    lse_join_lanes(z, lanes, a.k);
    bool bad;
    float tm = teacher_max(a, slot, at, li, lanes, bad);
    tm = lanes_most(tm, lanes);
    const bool any_bad = lanes_most(bad ? 1.f : 0.f, lanes) > 0.f;
    const bool has = tm != -kInf || any_bad;
    const float ts = lanes_total(teacher_sum(a, slot, at, li, lanes, tm), lanes);
    const float ls = __builtin_amdgcn_logf(z.s), lts = __builtin_amdgcn_logf(ts);
    float loss = 0.f;
    if (has) {
      loss = lanes_total(slots_loss(a, row, slot, at, li, lanes, z.m, ls, tm, lts), lanes);
      loss = any_bad ? __builtin_nanf("") : loss * (a.T * a.T * kLn2);
    }
    if (li == 0) {
      if (a.row_loss) a.row_loss[r] = loss;
      if (a.stat)
        *(float4*)(a.stat + 4 * r) = make_float4(z.m, ls, tm, lts);
      total += loss;
      some += has ? 1.f : 0.f;
    }
  }
  if (!a.part) return;
  if (li == 0) {
    red[0][grp] = total;
    red[1][grp] = some;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    float s = 0.f;
    for (int i = 0; i < groups; ++i) s += red[threadIdx.x][i];
    a.part[2 * blockIdx.x + threadIdx.x] = s;
  }
}

// Elements of a row before its first 16-byte boundary.
template <typename T>
__device__ inline int unaligned_head(const T* p, int n) {
  const int off = (int)(((uintptr_t)p & 15) / sizeof(T));
  return min(n, off ? (int)(16 / sizeof(T)) - off : 0);
}

__device__ inline float block_total(float v, float* red) {
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(1024) distill_block_kernel(DistillArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[16], red_m[16], red_s[16], red_t[16];
  const int tid = threadIdx.x, nt = blockDim.x;
  float total = 0.f, some = 0.f;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* row = (const T*)a.logits + r * a.ld;
    const int64_t at = r * a.K;
    const int head = unaligned_head(row, a.classes);
    const int chunks = (a.classes - head) / V, tail = head + chunks * V;
    const Slot slot(a, at, tid);
    Lse z;
    {
      float x[1] = {-kInf};
      if (tid < head) x[0] = (float)row[tid];
      else if (tid >= V && tid - V < a.classes - tail) x[0] = (float)row[tail + tid - V];
      if (tid < 2 * V) lse_add(z, x, a.k);
    }
    // kFlight accesses a lane in flight; the last turn's spare ones add -inf
    const T* body = row + head;
    for (int c = tid; c < chunks; c += kFlight * nt) {
      Pack<T, V> x[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        x[u] = *(const Pack<T, V>*)(body + (int64_t)min(c + u * nt, chunks - 1) * V);
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        if (c + u * nt >= chunks) break;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)x[u].v[i];
        lse_add(z, f, a.k);
      }
    }
    lse_join_lanes(z, 64, a.k);
    bool bad;
    float tm = lanes_most(teacher_max(a, slot, at, tid, nt, bad), 64);
    const float nbad = block_total(bad ? 1.f : 0.f, red);   // its barriers: the last
                                                            // row's readers of red_m, red_s, red_t
    if ((tid & 63) == 0) {
      red_m[tid >> 6] = z.m;
      red_s[tid >> 6] = z.s;
      red_t[tid >> 6] = tm;
    }
    __syncthreads();
    z = Lse{red_m[0], red_s[0]};
    tm = red_t[0];
    for (int i = 1; i < nt >> 6; ++i) {
      lse_join(z, red_m[i], red_s[i], a.k);
      tm = fmaxf(tm, red_t[i]);
    }
    const bool has = tm != -kInf || nbad > 0.f;
    const float ts = block_total(teacher_sum(a, slot, at, tid, nt, tm), red);
    const float ls = __builtin_amdgcn_logf(z.s), lts = __builtin_amdgcn_logf(ts);
    float loss = block_total(
        has ? slots_loss(a, row, slot, at, tid, nt, z.m, ls, tm, lts) : 0.f, red);
    loss = nbad > 0.f ? __builtin_nanf("") : loss * (a.T * a.T * kLn2);
    if (tid == 0) {
      if (a.row_loss) a.row_loss[r] = loss;
      if (a.stat)
        *(float4*)(a.stat + 4 * r) = make_float4(z.m, ls, tm, lts);
      total += loss;
      some += has ? 1.f : 0.f;
    }
  }
  if (tid == 0 && a.part) {
    a.part[2 * blockIdx.x] = total;
    a.part[2 * blockIdx.x + 1] = some;
  }
}

__global__ void __launch_bounds__(1024) distill_total_kernel(const float* part, int blocks,
                                                             float* total, int mean,
                                                             float* count) {
  __shared__ float red[16];
  float l = 0.f, n = 0.f;
  for (int i = threadIdx.x; i < blocks; i += 1024) {
    l += part[2 * i];
    n += part[2 * i + 1];
  }
  l = block_total(l, red);
  n = block_total(n, red);
  if (threadIdx.x == 0) {
    total[0] = mean ? l / fmaxf(n, 1.f) : l;
    count[0] = n;
  }
}

// The row's slots in LDS: class (-1: empty) and p. Returns whether a class is out of range.
__device__ inline bool stage_slots(const DistillArgs& a, const Slot& first, int64_t at, int li,
                                   int lanes, float tm, float lts, int* cls, float* ps) {
  bool bad = false;
  auto put = [&](int j, const Slot& s) {
    bad |= s.past();
    cls[j] = s.past() ? -1 : s.c;
    ps[j] = s.there() ? __builtin_amdgcn_exp2f((s.t - tm) * a.k - lts) : 0.f;
  };
  if (li < a.K) put(li, first);
  for (int j = li + lanes; j < a.K; j += lanes) put(j, Slot(a, at, j));
  return bad;
}
// The taught classes' gradients: the first slot of a class adds up all of its slots.
template <typename T>
__device__ inline void write_slots(const DistillArgs& a, const T* row, T* grad, int li, int lanes,
                                   float gi, float m, float ls, const int* cls, const float* ps) {
  for (int j = li; j < a.K; j += lanes) {
    const int c = cls[j];
    if (c < 0) continue;
    float p = 0.f;
    bool first = true;
    for (int i = 0; i < a.K; ++i)
      if (cls[i] == c) {
        p += ps[i];
        first &= i >= j;
      }
    if (first) grad[c] = (T)(gi * (__builtin_amdgcn_exp2f(((float)row[c] - m) * a.k - ls) - p));
  }
}
__device__ inline float row_factor(const DistillArgs& a, int64_t r) {
  float gi = a.g[r * a.g_stride] * a.T;
  if (a.count) gi /= fmaxf(*a.count, 1.f);
  return gi;
}

template <typename T>
__global__ void __launch_bounds__(256) distill_group_grad_kernel(DistillArgs a) {
  __shared__ int cls_lds[32 * kGroupSlots];
  __shared__ float p_lds[32 * kGroupSlots];
  const int lanes = a.lanes, li = threadIdx.x & (lanes - 1), grp = threadIdx.x / lanes;
  const int groups = 256 / lanes;
  int* cls = cls_lds + grp * kGroupSlots;
  float* ps = p_lds + grp * kGroupSlots;
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += (int64_t)gridDim.x * groups) {
    const int64_t r = r0 + grp;
    if (r >= a.rows) continue;
    const T* row = (const T*)a.logits + r * a.ld;
    T* grad = (T*)a.grad + r * a.classes;
    const Slot slot(a, r * a.K, li);
    float x[4];   // the first turn's logits, on their way before anything waits
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = (float)row[min(li + u * lanes, a.classes - 1)];
    const float4 st = *(const float4*)(a.stat + 4 * r);
    const bool has = st.w != -kInf;
    float gi = row_factor(a, r);
    bool bad = st.w != st.w;
    if (has) bad |= stage_slots(a, slot, r * a.K, li, lanes, st.z, st.w, cls, ps);
    if (lanes_most(bad ? 1.f : 0.f, lanes) > 0.f) gi = __builtin_nanf("");
    auto value = [&](float v) {
      return (T)(has ? gi * __builtin_amdgcn_exp2f((v - st.x) * a.k - st.y) : 0.f);
    };
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (li + u * lanes < a.classes) grad[li + u * lanes] = value(x[u]);
    for (int c = li + 4 * lanes; c < a.classes; c += lanes) grad[c] = value((float)row[c]);
    wave_lds_sync();   // the slots and the stores above, before this wave's next ones
    if (has) write_slots(a, row, grad, li, lanes, gi, st.x, st.y, cls, ps);
    wave_lds_sync();
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) distill_block_grad_kernel(DistillArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ int cls[kMaxSlots];
  __shared__ float ps[kMaxSlots];
  __shared__ float red[16];
  const int tid = threadIdx.x, nt = blockDim.x;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* row = (const T*)a.logits + r * a.ld;
    T* grad = (T*)a.grad + r * a.classes;
    const float4 st = *(const float4*)(a.stat + 4 * r);
    const bool has = st.w != -kInf;
    float gi = row_factor(a, r);
    const Slot slot(a, r * a.K, tid);
    __syncthreads();   // the last row's readers of the slots
    bool bad = st.w != st.w;
    if (has) bad |= stage_slots(a, slot, r * a.K, tid, nt, st.z, st.w, cls, ps);
    if (block_total(bad ? 1.f : 0.f, red) > 0.f) gi = __builtin_nanf("");
    auto value = [&](float x) {
      return has ? gi * __builtin_amdgcn_exp2f((x - st.x) * a.k - st.y) : 0.f;
    };
    const int head = unaligned_head(grad, a.classes);
    if (head == unaligned_head(row, a.classes)) {
      const int chunks = (a.classes - head) / V, tail = head + chunks * V;
      if (tid < head) grad[tid] = (T)value((float)row[tid]);
      if (tid < a.classes - tail) grad[tail + tid] = (T)value((float)row[tail + tid]);
      for (int c = tid; c < chunks; c += kFlight * nt) {
        Pack<T, V> x[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u)
          x[u] = *(const Pack<T, V>*)(row + head + (int64_t)min(c + u * nt, chunks - 1) * V);
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          if (c + u * nt >= chunks) break;
#pragma unroll
          for (int i = 0; i < V; ++i) x[u].v[i] = (T)value((float)x[u].v[i]);
          *(Pack<T, V>*)(grad + head + (int64_t)(c + u * nt) * V) = x[u];
        }
      }
    } else {   // rows of another alignment than the gradient's
      for (int c = tid; c < a.classes; c += nt) grad[c] = (T)value((float)row[c]);
    }
    __syncthreads();   // every store above is before the taught classes' own
    if (has) write_slots(a, row, grad, tid, nt, gi, st.x, st.y, cls, ps);
  }
}

bool group_form(int64_t classes, int K) { return classes <= kGroupClasses && K <= kGroupSlots; }
int group_lanes(int64_t classes) {
  int l = 8;
  while (l < 64 && l * 4 < classes) l <<= 1;
  return l;
}
int distill_blocks(int64_t rows, int64_t classes, int K) {
  const int64_t per = group_form(classes, K) ? 256 / group_lanes(classes) : 1;
  return (int)std::min<int64_t>(ceil_div(rows, per), kMaxBlocks);
}
// A workgroup a row: few rows leave CUs to themselves, so each gets all the lanes it can have. Else 256
// (forward) or 512 lanes: 8192 x 32000 bf16, forward 159 / 173 / 273 us with 256 / 512 / 1024, backward
// 214 / 202 / 241 us. (A plain read of the logits runs in 140 us, their copy in 205.)
int block_threads(int64_t rows, bool backward) {
  return rows < 512 ? 1024 : backward ? 512 : 256;
}

int check_distill(const char* what, int dtype, int64_t rows, int64_t classes, int teacher_dtype,
                  int K, float temperature) {
  GATX_REQUIRE(dtype_ok(dtype) && dtype_ok(teacher_dtype), "%s: unknown dtype", what);
  GATX_REQUIRE(rows >= 0 && classes >= 1 && classes < (1ll << 30), "%s: %lld x %lld logits", what,
               (long long)rows, (long long)classes);
  GATX_REQUIRE(K >= 1 && K <= kMaxSlots, "%s: %d slots a row (1..%d)", what, K, kMaxSlots);
  GATX_REQUIRE(temperature > 9e-19f && temperature < 1.1e18f,   // T^2 and 1 / T are float32 numbers
               "%s: temperature must be positive (1e-18 to 1e18)", what);
  return 0;
}

}  // namespace
}  // namespace gatx

using namespace gatx;

extern "C" size_t gatx_topk_distill_workspace_bytes(int64_t rows) {
  return sizeof(float) * 2 * (size_t)std::min<int64_t>(std::max<int64_t>(rows, 1), kMaxBlocks);
}

extern "C" int gatx_topk_distill(int dtype, const void* logits, int64_t rows, int64_t classes,
                                 int64_t ld, int teacher_dtype, const void* teacher,
                                 const void* index, int index_is_int64, int K, float temperature,
                                 float* row_loss, float* total, int mean, float* count,
                                 float* stat, void* workspace, size_t workspace_bytes, gatx_stream_t s) {
  GATX_CALL(check_distill("topk_distill", dtype, rows, classes, teacher_dtype, K, temperature));
  hipStream_t st = (hipStream_t)s;
  GATX_REQUIRE(!total || count, "topk_distill: null count");
  if (rows == 0) {
    if (total) {
      zero_words_kernel<<<1, 64, 0, st>>>((uint32_t*)total, 1);
      zero_words_kernel<<<1, 64, 0, st>>>((uint32_t*)count, 1);
    }
    GATX_LAUNCH_CHECK("topk_distill zero");
    return 0;
  }
  GATX_REQUIRE(logits && teacher && index, "topk_distill: null input");
  GATX_REQUIRE(!total || (workspace && workspace_bytes >= gatx_topk_distill_workspace_bytes(rows)),
               "topk_distill: workspace too small");
  DistillArgs a = {};
  a.logits = logits; a.teacher = teacher; a.index = index; a.rows = rows; a.ld = ld;
  a.classes = (int)classes; a.K = K; a.teacher_dtype = teacher_dtype; a.index64 = index_is_int64;
  a.T = temperature; a.k = kLog2e / temperature;
  a.row_loss = row_loss; a.part = total ? (float*)workspace : nullptr; a.stat = stat;
  a.lanes = group_lanes(classes);
  const int blocks = distill_blocks(rows, classes, K);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (group_form(classes, K)) distill_group_kernel<T><<<blocks, 256, 0, st>>>(a);
    else distill_block_kernel<T><<<blocks, block_threads(rows, false), 0, st>>>(a);
    return 0;
  });
  GATX_LAUNCH_CHECK("topk_distill");
  if (total) {
    distill_total_kernel<<<1, 1024, 0, st>>>((const float*)workspace, blocks, total, mean,
                                            count);
    GATX_LAUNCH_CHECK("topk_distill_total");
  }
  return 0;
}

extern "C" int gatx_topk_distill_backward(int dtype, const void* logits, int64_t rows,
                                          int64_t classes, int64_t ld, int teacher_dtype,
                                          const void* teacher, const void* index,
                                          int index_is_int64, int K, float temperature,
                                          const float* stat, const float* g, int g_stride,
                                          const float* count, void* grad, gatx_stream_t s) {
  GATX_CALL(check_distill("topk_distill_backward", dtype, rows, classes, teacher_dtype, K,
                          temperature));
  if (rows == 0) return 0;
  GATX_REQUIRE(logits && teacher && index && stat && g && grad,
               "topk_distill_backward: null buffer");
  GATX_REQUIRE(g_stride == 0 || g_stride == 1, "topk_distill_backward: g_stride is 0 or 1");
  DistillArgs a = {};
  a.logits = logits; a.teacher = teacher; a.index = index; a.rows = rows; a.ld = ld;
  a.classes = (int)classes; a.K = K; a.teacher_dtype = teacher_dtype; a.index64 = index_is_int64;
  a.T = temperature; a.k = kLog2e / temperature;
  a.stat = const_cast<float*>(stat); a.g = g; a.count = count; a.g_stride = g_stride;
  a.grad = grad; a.lanes = group_lanes(classes);
  hipStream_t st = (hipStream_t)s;
  // every row's work is its own: as many workgroups as rows fill, no fixed walk to keep
  const int64_t per = group_form(classes, K) ? 256 / a.lanes : 1;
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(rows, per), 1 << 20);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (group_form(classes, K)) distill_group_grad_kernel<T><<<blocks, 256, 0, st>>>(a);
    else distill_block_grad_kernel<T><<<blocks, block_threads(rows, true), 0, st>>>(a);
    return 0;
  });
  GATX_LAUNCH_CHECK("topk_distill_backward");
  return 0;
}
