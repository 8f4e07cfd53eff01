// Distillation from a teacher's top logits (gpn_distill_forward, _backward, _step) for gfx950.
//
//   p = softmax over the K entries of t / T;  ls_c = z_c / T - log sum_c' exp(z_c' / T)
//   loss = T^2 w sum_k p_k (log p_k - ls_{idx_k});   d loss / dz_c = w T (exp(ls_c) - sum_{k: idx_k = c} p_k)
//
// Bound by the logits' bytes: read once, and their gradient written once.  Two layouts:
//   rows    classes are contiguous (a large vocabulary): one workgroup per row.  The row stays in registers between the pass
//           that finds its maximum and sum and the pass that writes the gradient, so the step kernel reads it once.
//   planes  rows are contiguous (class planes of an image): one lane per row, every class a coalesced read.
// Maxima, sums and gradients are fp32 and rounded once at the store.  Every row's work is done by one workgroup in a fixed order,
// and the sum over the rows by one workgroup: no atomic, the same bits every time.
#include <climits>

#include "common.h"

namespace {

typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef unsigned short bfu;  // bf16 bits

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

struct DistP {
  const void *z, *t, *idx;
  void* dz;
  long long z_rs, z_cs, t_rs, t_ks, i_rs, i_ks, d_rs, d_cs;
  const float *w, *dloss, *lse_in;
  float *loss_rows, *lse;
  long long N;
  int C, K, t_f32, i_64, dloss_rows;
  float T, c;        // temperature, log2(e) / T
  float grad_scale;  // of the upstream gradient (1 / N for a mean)
  float loss_scale;  // of the sum over the rows
};

__device__ __forceinline__ float bf2f(unsigned x) { return __builtin_bit_cast(float, x << 16); }
__device__ __forceinline__ bfu f2bf(float x) { return __builtin_bit_cast(bfu, (__bf16)x); }

template <typename T>
struct El;
template <>
struct El<float> {
  static constexpr int EP = 4;
  static constexpr unsigned NEG = 0xff800000u;  // -inf
  static __device__ __forceinline__ float get(const u4v& r, int i) { return __builtin_bit_cast(float, (unsigned)r[i]); }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float x) { *p = x; }
  static __device__ __forceinline__ u4v pack(const float* x) {
    u4v r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, x[i]);
    return r;
  }
  static __device__ __forceinline__ u4v gather(const float* p, int lo, int hi) {  // elements lo .. hi-1 of a chunk, others -inf
    u4v r = {NEG, NEG, NEG, NEG};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i >= lo && i < hi) r[i] = __builtin_bit_cast(unsigned, p[i]);
    return r;
  }
};
template <>
struct El<bfu> {
  static constexpr int EP = 8;
  static constexpr unsigned NEG = 0xff80ff80u;
  static __device__ __forceinline__ float get(const u4v& r, int i) {
    return __builtin_bit_cast(float, i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  }
  static __device__ __forceinline__ float load(const bfu* p) { return bf2f(*p); }
  static __device__ __forceinline__ void store(bfu* p, float x) { *p = f2bf(x); }
  static __device__ __forceinline__ u4v pack(const float* x) {
    u4v r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (unsigned)f2bf(x[2 * i]) | (unsigned)f2bf(x[2 * i + 1]) << 16;
    return r;
  }
  static __device__ __forceinline__ u4v gather(const bfu* p, int lo, int hi) {
    u4v r = {NEG, NEG, NEG, NEG};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= lo && i < hi) {
        const unsigned x = p[i];
        r[i >> 1] = i & 1 ? (r[i >> 1] & 0xffffu) | x << 16 : (r[i >> 1] & 0xffff0000u) | x;
      }
    return r;
  }
};

// Entry k of a row: its class, or -1 where the entry is left out (outside [0, C)); its logit.
__device__ __forceinline__ int entry_class(const DistP& a, long long row, int k) {
  const long long at = row * a.i_rs + (long long)k * a.i_ks;
  const long long x = a.i_64 ? ((const long long*)a.idx)[at] : ((const int*)a.idx)[at];
  return x >= 0 && x < a.C ? (int)x : -1;
}
__device__ __forceinline__ float entry_logit(const DistP& a, long long row, int k) {
  const long long at = row * a.t_rs + (long long)k * a.t_ks;
  return a.t_f32 ? ((const float*)a.t)[at] : bf2f(((const bfu*)a.t)[at]);
}

enum { FWD = 0, BWD = 1, STEP = 2 };

// What exponentials are taken relative to: the maximum, or 0 where that is infinite (nothing seen yet, or a value of +inf).
__device__ __forceinline__ float base_of(float m) { return fabsf(m) == INFINITY ? 0.f : m; }

// Combination of two (maximum, sum relative to it).
__device__ __forceinline__ void merge(float& m, float& l, float m2, float l2, float c) {
  const float M = fmaxf(m, m2), s = base_of(M);
  l = l * exp2_((m - s) * c) + l2 * exp2_((m2 - s) * c);
  m = M;
}

// gradient's factor of a row
__device__ __forceinline__ float row_factor(const DistP& a, long long row) {
  const float g = a.dloss ? a.dloss[a.dloss_rows ? row : 0] : 1.f;
  return g * a.grad_scale * a.T * (a.w ? a.w[row] : 1.f);
}

// ---------------------------------------------------------------------------------------------------------- rows
// NT threads, CH 16-byte chunks of the row in each thread's registers; a row of more than NT * CH chunks is walked in segments
// and read again for the gradient.
template <typename T, int NT, int CH, int MODE>
__global__ void __launch_bounds__(NT) k_distill_rows(const DistP a) {
  using E = El<T>;
  constexpr int EP = E::EP, NW = NT / 64;
  __shared__ float sp[GPN_DISTILL_MAX_K], sred[2 * NW], sstat[4];
  __shared__ int si[GPN_DISTILL_MAX_K];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* z = (const T*)a.z + row * a.z_rs;
  const int a0 = (int)(((size_t)z & 15) / sizeof(T));  // elements of the first chunk before the row
  const int nch = (int)(((long long)a0 + a.C + EP - 1) / EP);
  const T* zc = z - a0;

  u4v r[CH];
  const auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = c0 + tid + i * NT;
      r[i] = u4v{E::NEG, E::NEG, E::NEG, E::NEG};
      if (c < nch) {
        const long long e = (long long)c * EP;
        const int lo = c == 0 ? a0 : 0;
        const long long left = a.C + a0 - e;
        if (lo == 0 && left >= EP) r[i] = *(const u4v*)(zc + e);
        else r[i] = E::gather(zc + e, lo, left < EP ? (int)left : EP);
      }
    }
  };
  const int seg = NT * CH;
  load(0);

  // teacher: wave 0 walks the K entries while the row is on its way
  if (wave == 0) {
    float mt = -INFINITY, lt = 0.f;
    for (int k = lane; k < a.K; k += 64) {
      const int x = entry_class(a, row, k);
      const float t = x >= 0 ? entry_logit(a, row, k) : -INFINITY;
      si[k] = x, sp[k] = t;
      const float M = fmaxf(mt, t), s = base_of(M);
      lt = lt * exp2_((mt - s) * a.c) + exp2_((t - s) * a.c);
      mt = M;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) merge(mt, lt, __shfl_xor(mt, d), __shfl_xor(lt, d), a.c);
    if (lane == 0) sstat[0] = mt, sstat[1] = lt;
  }

  float m = -INFINITY, l = 0.f;
  if (MODE != BWD) {
    for (int c0 = 0;;) {
      float mx = m;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < EP; ++e) mx = fmaxf(mx, E::get(r[i], e));
      const float s = base_of(mx);
      l *= exp2_((m - s) * a.c);
      m = mx;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < EP; ++e) l += exp2_((E::get(r[i], e) - s) * a.c);
      c0 += seg;
      if (c0 >= nch) break;
      load(c0);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) merge(m, l, __shfl_xor(m, d), __shfl_xor(l, d), a.c);
    if (lane == 0) sred[wave] = m, sred[NW + wave] = l;
  }
  __syncthreads();
  if (MODE != BWD) {
    m = sred[0], l = sred[NW];
#pragma unroll
    for (int w = 1; w < NW; ++w) merge(m, l, sred[w], sred[NW + w], a.c);
  }
  const float mt = sstat[0], lt = sstat[1];
  const bool empty = !(lt > 0.f) && lt == lt;  // no entry at all
  const float lt2 = log2_(lt);
  // log2 of the student's probability of a logit x: (x - m) c - l2
  float l2;
  if (MODE == BWD) m = 0.f, l2 = a.lse_in[row] * LOG2E;
  else l2 = log2_(l);
  if (MODE != BWD && wave == 0) {
    float loss = 0.f;
    for (int k = lane; k < a.K; k += 64) {
      const int x = si[k];
      const float lp = (sp[k] - mt) * a.c - lt2, p = exp2_(lp);
      if (x >= 0 && !(p == 0.f)) loss += p * (lp - ((E::load(z + x) - m) * a.c - l2));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) loss += __shfl_xor(loss, d);
    if (lane == 0) {
      a.loss_rows[row] = empty ? 0.f : loss * LN2 * a.T * a.T * (a.w ? a.w[row] : 1.f);
      if (MODE == FWD) a.lse[row] = (m * a.c + l2) * LN2;
    }
  }
  if (MODE == FWD) return;

  const float f = row_factor(a, row);
  T* dz = (T*)a.dz + row * a.d_rs;
  const bool same = (((size_t)dz ^ (size_t)z) & 15) == 0;  // 16-byte stores meet 16-byte loads
  const float inv = MODE == BWD ? 0.f : 1.f / l;
  for (int c0 = 0; c0 < nch; c0 += seg) {
    if (nch > seg && (MODE == BWD ? c0 > 0 : true)) load(c0);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = c0 + tid + i * NT;
      if (c < nch) {
        float y[EP];
#pragma unroll
        for (int e = 0; e < EP; ++e) {
          const float x = (E::get(r[i], e) - m) * a.c;
          const float s = MODE == BWD ? exp2_(x - l2) : exp2_(x) * inv;
          y[e] = empty ? 0.f : f * s;
        }
        const long long at = (long long)c * EP - a0;
        const int lo = c == 0 ? a0 : 0;
        const long long left = a.C - at;
        if (same && lo == 0 && left >= EP) {
          *(u4v*)(dz + at) = E::pack(y);
        } else {
#pragma unroll
          for (int e = 0; e < EP; ++e)
            if (e >= lo && e < left) E::store(dz + at + e, y[e]);
        }
      }
    }
  }
  if (empty) return;
  // The teacher's classes: their entries are written a second time, behind the barrier.  A class that stands in the row twice
  // has both probabilities in its sum, in the order of the entries, whichever of the two writes it.
  __threadfence_block();
  __syncthreads();
  for (int k = tid; k < a.K; k += NT) {
    const int x = si[k];
    if (x < 0) continue;
    float p = 0.f;
    for (int j = 0; j < a.K; ++j)
      if (si[j] == x) p += exp2_((sp[j] - mt) * a.c - lt2);
    const float u = (E::load(z + x) - m) * a.c, s = MODE == BWD ? exp2_(u - l2) : exp2_(u) * inv;
    E::store(dz + x, f * (s - p));
  }
}

// -------------------------------------------------------------------------------------------------------- planes
// One lane per row; with C <= CM the classes stay in registers.
template <typename T, int CM, int MODE>
__global__ void __launch_bounds__(256) k_distill_planes(const DistP a) {
  using E = El<T>;
  const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.N) return;
  const T* z = (const T*)a.z + row;
  float x[CM > 0 ? CM : 1];
  float m = -INFINITY, l = 0.f;
  if (CM > 0) {
#pragma unroll
    for (int c = 0; c < CM; ++c) x[c] = c < a.C ? E::load(z + c * a.z_cs) : -INFINITY;
  }
  if (MODE != BWD) {
    if (CM > 0) {
#pragma unroll
      for (int c = 0; c < CM; ++c) m = fmaxf(m, x[c]);
      const float s = base_of(m);
#pragma unroll
      for (int c = 0; c < CM; ++c) l += exp2_((x[c] - s) * a.c);
    } else {
      for (int c = 0; c < a.C; ++c) {
        const float v = E::load(z + c * a.z_cs), M = fmaxf(m, v), s = base_of(M);
        l = l * exp2_((m - s) * a.c) + exp2_((v - s) * a.c);
        m = M;
      }
    }
  }
  float mt = -INFINITY, lt = 0.f;
  for (int k = 0; k < a.K; ++k) {
    const float t = entry_class(a, row, k) >= 0 ? entry_logit(a, row, k) : -INFINITY;
    const float M = fmaxf(mt, t), s = base_of(M);
    lt = lt * exp2_((mt - s) * a.c) + exp2_((t - s) * a.c);
    mt = M;
  }
  const bool empty = !(lt > 0.f) && lt == lt;
  const float lt2 = log2_(lt);
  float l2;
  if (MODE == BWD) m = 0.f, l2 = a.lse_in[row] * LOG2E;
  else l2 = log2_(l);
  if (MODE != BWD) {
    float loss = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int cl = entry_class(a, row, k);
      if (cl < 0) continue;
      const float lp = (entry_logit(a, row, k) - mt) * a.c - lt2, p = exp2_(lp);
      if (!(p == 0.f)) loss += p * (lp - ((E::load(z + cl * a.z_cs) - m) * a.c - l2));
    }
    a.loss_rows[row] = empty ? 0.f : loss * LN2 * a.T * a.T * (a.w ? a.w[row] : 1.f);
    if (MODE == FWD) a.lse[row] = (m * a.c + l2) * LN2;
  }
  if (MODE == FWD) return;
  const float f = row_factor(a, row), inv = MODE == BWD ? 0.f : 1.f / l;
  const auto grad = [&](float v) {
    const float u = (v - m) * a.c;
    return MODE == BWD ? exp2_(u - l2) : exp2_(u) * inv;
  };
  T* dz = (T*)a.dz + row;
  if (CM > 0) {
#pragma unroll
    for (int c = 0; c < CM; ++c)
      if (c < a.C) E::store(dz + c * a.d_cs, empty ? 0.f : f * grad(x[c]));
  } else {
    for (int c = 0; c < a.C; ++c) E::store(dz + c * a.d_cs, empty ? 0.f : f * grad(E::load(z + c * a.z_cs)));
  }
  if (empty) return;
  for (int k = 0; k < a.K; ++k) {  // the teacher's classes again, by the lane that wrote them
    const int cl = entry_class(a, row, k);
    if (cl < 0) continue;
    float p = 0.f;
    for (int j = 0; j < a.K; ++j)
      if (entry_class(a, row, j) == cl) p += exp2_((entry_logit(a, row, j) - mt) * a.c - lt2);
    E::store(dz + cl * a.d_cs, f * (grad(E::load(z + cl * a.z_cs)) - p));
  }
}

// Sum of the rows' losses by one workgroup, in 64 bits.
__global__ void __launch_bounds__(1024) k_distill_sum(const float* __restrict__ rows, long long N, float scale, float* __restrict__ out) {
  __shared__ double part[16];
  double s = 0.;
  for (long long i = threadIdx.x; i < N; i += 1024) s += rows[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.;
    for (int w = 0; w < 16; ++w) s += part[w];
    *out = (float)(s * (double)scale);
  }
}

// ----------------------------------------------------------------------------------------------------------- host
template <typename T, int MODE>
void launch_rows(const DistP& a, hipStream_t st) {
  // Threads by the length of the row: a wave where that gives each lane at most 4 chunks, then workgroups of 256 and 1024.
  const long long nch = ((long long)a.C + El<T>::EP - 1) / El<T>::EP + 1;
  const dim3 grid((unsigned)a.N);
#define GPN_ROWS(NT, CH) hipLaunchKernelGGL((k_distill_rows<T, NT, CH, MODE>), grid, dim3(NT), 0, st, a)
  if (nch <= 64) GPN_ROWS(64, 1);
  else if (nch <= 256) GPN_ROWS(64, 4);
  else if (nch <= 1024) GPN_ROWS(256, 4);
  else if (nch <= 2048) GPN_ROWS(256, 8);
  else if (nch <= 4096) GPN_ROWS(1024, 4);
  else if (nch <= 8192) GPN_ROWS(1024, 8);
  else GPN_ROWS(1024, 16);
#undef GPN_ROWS
}

template <typename T, int MODE>
void launch_planes(const DistP& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.N + 255) / 256));
  if (a.C <= 32) hipLaunchKernelGGL((k_distill_planes<T, 32, MODE>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_distill_planes<T, 0, MODE>), grid, dim3(256), 0, st, a);
}

template <int MODE>
int run(const gpn_distill_args_t* x, hipStream_t st, const char* name) {
  GPN_REQUIRE(x, "%s: null arguments", name);
  GPN_REQUIRE(x->dtype == GPN_DT_F32 || x->dtype == GPN_DT_BF16, "%s: unknown dtype %d", name, x->dtype);
  GPN_REQUIRE(x->teacher_dtype == GPN_DT_F32 || x->teacher_dtype == GPN_DT_BF16, "%s: unknown teacher dtype %d", name, x->teacher_dtype);
  GPN_REQUIRE(x->index_bytes == 4 || x->index_bytes == 8, "%s: indices of %d bytes", name, x->index_bytes);
  GPN_REQUIRE(x->N >= 0 && x->N <= INT_MAX, "%s: %lld rows", name, x->N);
  GPN_REQUIRE(x->C >= 1 && x->C <= (1 << 30), "%s: %d classes", name, x->C);
  GPN_REQUIRE(x->K >= 0 && x->K <= GPN_DISTILL_MAX_K, "%s: K must be in [0,%d] (got %d)", name, GPN_DISTILL_MAX_K, x->K);
  GPN_REQUIRE(x->temperature > 0.f && x->temperature < INFINITY, "%s: temperature must be positive and finite", name);
  GPN_REQUIRE(x->reduction >= GPN_RED_NONE && x->reduction <= GPN_RED_MEAN, "%s: unknown reduction %d", name, x->reduction);
  GPN_REQUIRE(x->logits || x->N == 0, "%s: null logits", name);
  GPN_REQUIRE((x->teacher && x->index) || x->K == 0 || x->N == 0, "%s: null teacher", name);
  const bool planes = x->class_stride != 1 && x->C > 1;
  GPN_REQUIRE(!planes || x->row_stride == 1 || x->N <= 1, "%s: logits need contiguous classes or contiguous rows (strides %lld, %lld)",
              name, x->row_stride, x->class_stride);
  if (MODE != BWD) {
    GPN_REQUIRE(x->loss_rows || x->N == 0, "%s: null loss_rows", name);
    GPN_REQUIRE(x->loss || x->reduction == GPN_RED_NONE, "%s: null loss", name);
  }
  if (MODE != STEP) GPN_REQUIRE(x->lse || x->N == 0, "%s: null lse", name);
  if (MODE == BWD) GPN_REQUIRE(x->dloss || x->N == 0, "%s: null dloss", name);
  if (MODE != FWD) {
    GPN_REQUIRE(x->dlogits || x->N == 0, "%s: null dlogits", name);
    GPN_REQUIRE(planes ? x->drow_stride == 1 || x->N <= 1 : x->dclass_stride == 1 || x->C == 1,
                "%s: dlogits must lie as the logits do", name);
  }
  DistP a = {};
  a.z = x->logits, a.t = x->teacher, a.idx = x->index, a.dz = x->dlogits;
  a.z_rs = x->row_stride, a.z_cs = x->class_stride, a.t_rs = x->teacher_stride[0], a.t_ks = x->teacher_stride[1];
  a.i_rs = x->index_stride[0], a.i_ks = x->index_stride[1], a.d_rs = x->drow_stride, a.d_cs = x->dclass_stride;
  a.w = x->row_weight, a.loss_rows = x->loss_rows, a.lse = x->lse, a.lse_in = x->lse;
  a.dloss = MODE == BWD ? x->dloss : nullptr, a.dloss_rows = x->reduction == GPN_RED_NONE;
  a.N = x->N, a.C = x->C, a.K = x->K, a.t_f32 = x->teacher_dtype == GPN_DT_F32, a.i_64 = x->index_bytes == 8;
  a.T = x->temperature, a.c = LOG2E / x->temperature;
  const float mean = x->reduction == GPN_RED_MEAN && x->N > 0 ? 1.f / (float)x->N : 1.f;
  a.grad_scale = mean * (MODE == STEP ? x->grad_scale : 1.f);
  if (x->N > 0) {
    if (x->dtype == GPN_DT_F32) planes ? launch_planes<float, MODE>(a, st) : launch_rows<float, MODE>(a, st);
    else planes ? launch_planes<bfu, MODE>(a, st) : launch_rows<bfu, MODE>(a, st);
    GPN_LAUNCH_CHECK(name);
  }
  if (MODE != BWD && x->reduction != GPN_RED_NONE) {
    hipLaunchKernelGGL(k_distill_sum, dim3(1), dim3(1024), 0, st, x->loss_rows, x->N, mean, x->loss);
    GPN_LAUNCH_CHECK("k_distill_sum");
  }
  return GPN_OK;
}

}  // namespace

extern "C" int gpn_distill_forward(const gpn_distill_args_t* a, gpn_stream_t stream) {
  return run<FWD>(a, (hipStream_t)stream, "gpn_distill_forward");
}
extern "C" int gpn_distill_backward(const gpn_distill_args_t* a, gpn_stream_t stream) {
  return run<BWD>(a, (hipStream_t)stream, "gpn_distill_backward");
}
extern "C" int gpn_distill_step(const gpn_distill_args_t* a, gpn_stream_t stream) {
  return run<STEP>(a, (hipStream_t)stream, "gpn_distill_step");
}
