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
  int C, K, t_f32, i_64, dloss_rows, loss_each;  // loss_each: loss_rows is an output (else workgroups may leave sums there)
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
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    b8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)x[i];
    return __builtin_bit_cast(u4v, r);
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

// Backward: whether a row's probabilities are formed from its stored log-sum-exp (given in powers of two).  Up to 32 of them half a
// step of fp32 is 2^-20, about what the row's sum is off by itself; beyond, a common offset of the logits would drown their
// differences, and the row's maximum and sum are formed once more (4096 x 48000 bf16: 184 us where every row is such a one, 175 where
// none is; 500 x 140000 bf16, read a second time for it: 83 and 54).
__device__ __forceinline__ bool lse_serves(float l2) { return fabsf(l2) <= 32.f; }

// log sum exp(z / T) from the maximum and log2 of the sum relative to it.  (m c alone would overflow for logits near the type's
// limits, whose log-sum-exp is a number.)
__device__ __forceinline__ float row_lse(const DistP& a, float m, float l2) { return m / a.T + l2 * LN2; }

// gradient's factor of a row of weight w
__device__ __forceinline__ float row_factor(const DistP& a, long long row, float w) {
  const float g = a.dloss ? a.dloss[a.dloss_rows ? row : 0] : 1.f;
  return g * a.grad_scale * a.T * w;
}

// ---------------------------------------------------------------------------------------------------------- rows
// NT threads, CH 16-byte chunks of the row in each thread's registers.  MANY: a row of more than NT * CH chunks is walked in
// segments and read again for the gradient.  The elements before the first and behind the last 16-byte boundary of the row
// belong to the first 2 EP threads, one each.
// The step, read and write together: 4096 x 48000 bf16 185 us, 4.2 TB/s (a large copy: 4.8); 1000 x 65000 fp32 113 us, 4.6; 257 x 10007
// fp32, not one row in 256 on a boundary, 10 us.
template <typename T, int NT, int CH, bool MANY, int MODE>
__global__ void __launch_bounds__(NT, CH > 8 ? 4 : 6) k_distill_rows(const DistP a) {
  using E = El<T>;
  constexpr int EP = E::EP, NW = NT / 64;
  __shared__ float sp[GPN_DISTILL_MAX_K], sred[2 * NW], sstat[2];
  __shared__ int si[GPN_DISTILL_MAX_K];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* z = (const T*)a.z + row * a.z_rs;
  const int a0 = (int)(((size_t)z & 15) / sizeof(T));  // elements of the first chunk before the row
  const int head = min(a0 ? EP - a0 : 0, a.C), nch = (a.C - head) / EP;  // then nch whole chunks from zc
  const T* zc = z + head;
  // the thread's own element at an end of the row (or none): head elements, then those behind the last chunk
  const int edge = tid < head ? tid : tid >= EP && tid < 2 * EP && head + nch * EP + tid - EP < a.C ? head + nch * EP + tid - EP : -1;
  const float xe = edge >= 0 ? E::load(z + edge) : -INFINITY;

  u4v r[CH];
  int at = tid;  // opaque below: addresses are formed again for every pass rather than held over it
  const auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = c0 + at + i * NT;
      r[i] = u4v{E::NEG, E::NEG, E::NEG, E::NEG};
      if (c < nch) r[i] = *(const u4v*)((const char*)zc + (unsigned)c * 16u);
    }
  };
  // unpack again rather than hold the row a second time, in fp32
  const auto again = [&]() {
#pragma unroll
    for (int i = 0; i < CH; ++i) asm volatile("" : "+v"(r[i]));
    asm volatile("" : "+v"(at));
  };
  constexpr int seg = NT * CH;
  load(0);

  // teacher: wave 0 walks the K entries while the row is on its way
  if (wave == 0) {
    float mt = -INFINITY, lt = 0.f;
    for (int k = lane; k < a.K; k += 64) {
      const int x = entry_class(a, row, k);
      const float t = x >= 0 ? entry_logit(a, row, k) : -INFINITY;
      si[k] = x, sp[k] = t;
      merge(mt, lt, t, 1.f, a.c);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) merge(mt, lt, __shfl_xor(mt, d), __shfl_xor(lt, d), a.c);
    if (lane == 0) sstat[0] = mt, sstat[1] = lt;
  }

  // log2 of a logit's probability: (x - m) c - l2.  The difference comes first: x c - m c of logits of 10^9 would be noise.
  float l2 = MODE == BWD ? a.lse_in[row] * LOG2E : 0.f;
  const bool walk = MODE != BWD || !lse_serves(l2);
  float m = xe, l = fabsf(xe) == INFINITY ? exp2_(xe) : edge >= 0 ? exp2_((xe - base_of(xe)) * a.c) : 0.f;
  if (walk) {
    if constexpr (MANY && MODE == BWD) {
      // The first segment stays in its registers: a chunk at a time, so that no more of them are taken than for the gradient alone
      // and two workgroups fit a CU (500 x 140000 bf16, rows whose stored value serves: 54 us, 59 with the loop below).
#pragma unroll 1
      for (int c = tid; c < nch; c += NT) {
        const u4v y = *(const u4v*)((const char*)zc + (unsigned)c * 16u);
        float mx = m;
#pragma unroll
        for (int e = 0; e < EP; ++e) mx = fmaxf(mx, E::get(y, e));
        const float b = base_of(mx);
        l *= exp2_((m - b) * a.c);
        m = mx;
#pragma unroll
        for (int e = 0; e < EP; ++e) l += exp2_((E::get(y, e) - b) * a.c);
      }
    }
    for (int c0 = 0; !(MANY && MODE == BWD);) {
      float mx = m;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (c0 + i * NT < nch) {
#pragma unroll
          for (int e = 0; e < EP; ++e) mx = fmaxf(mx, E::get(r[i], e));
        }
      const float b = base_of(mx);
      l *= exp2_((m - b) * a.c);
      m = mx;
      again();
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (c0 + i * NT < nch) {
#pragma unroll
          for (int e = 0; e < EP; ++e) l += exp2_((E::get(r[i], e) - b) * a.c);
        }
      c0 += seg;
      if (!MANY || c0 >= nch) break;
      load(c0);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) merge(m, l, __shfl_xor(m, d), __shfl_xor(l, d), a.c);
    if (lane == 0) sred[wave] = m, sred[NW + wave] = l;
  }
  __syncthreads();
  if (walk) {
    m = sred[0], l = sred[NW];
#pragma unroll
    for (int w = 1; w < NW; ++w) merge(m, l, sred[w], sred[NW + w], a.c);
    l2 = log2_(l);
  } else {
    m = 0.f;
  }
  const float mt = sstat[0], lt = sstat[1];
  const float wt = a.w ? a.w[row] : 1.f;
  const bool empty = wt == 0.f || (!(lt > 0.f) && lt == lt);  // left out, or no entry at all
  const float lt2 = log2_(lt);
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
      a.loss_rows[row] = empty ? 0.f : loss * LN2 * a.T * a.T * wt;
      if (MODE == FWD) a.lse[row] = row_lse(a, m, l2);
    }
  }
  if (MODE == FWD) return;

  const float f = row_factor(a, row, wt);
  const float inv = MODE == BWD ? 0.f : 1.f / l, fi = f * inv;
  const auto prob = [&](float x) {
    const float u = (x - m) * a.c;
    return MODE == BWD ? exp2_(u - l2) : exp2_(u) * inv;
  };
  T* dz = (T*)a.dz + row * a.d_rs;
  if (empty) {  // zero whatever the logits hold
    for (int c = tid; c < a.C; c += NT) E::store(dz + c, 0.f);
    return;
  }
  const auto grad = [&](float x) {
    const float u = (x - m) * a.c;
    return MODE == BWD ? f * exp2_(u - l2) : fi * exp2_(u);
  };
  if (edge >= 0) E::store(dz + edge, grad(xe));
  const bool same = (((size_t)dz ^ (size_t)z) & 15) == 0;  // 16-byte stores meet 16-byte loads
  for (int c0 = 0; c0 < nch; c0 += seg) {
    again();
    if (MANY && (MODE == BWD ? c0 > 0 : true)) load(c0);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = c0 + at + i * NT;
      if (c < nch) {
        float y[EP];
#pragma unroll
        for (int e = 0; e < EP; ++e) y[e] = grad(E::get(r[i], e));
        T* d = (T*)((char*)(dz + head) + (unsigned)c * 16u);
        if (same) {
          *(u4v*)d = E::pack(y);
        } else {
#pragma unroll
          for (int e = 0; e < EP; ++e) E::store(d + e, y[e]);
        }
      }
    }
  }
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
    E::store(dz + x, f * (prob(E::load(z + x)) - p));
  }
}

// -------------------------------------------------------------------------------------------------------- planes
// VEC neighbouring rows per lane.  With C <= CM the classes stay in registers, else they are walked twice in blocks of 8; with
// K <= KM so do the teacher's entries (their addresses differ from lane to lane: all are requested at once).
// The step of 300000 x 150 bf16, 8 entries: 112 us, 1.6 TB/s and the entries' 24 MB; of a 240 x 320 image of 21 fp32 classes, 5
// entries: 11 us, 1.2 TB/s, as long as its longest chain of loads takes.
template <typename T, int VEC>
struct Px;
template <>
struct Px<float, 1> {
  float r;
  __device__ __forceinline__ void load(const float* p) { r = *p; }
  __device__ __forceinline__ float get(int) const { return r; }
  static __device__ __forceinline__ void store(float* p, const float* y) { *p = y[0]; }
};
template <>
struct Px<bfu, 1> {
  bfu r;
  __device__ __forceinline__ void load(const bfu* p) { r = *p; }
  __device__ __forceinline__ float get(int) const { return bf2f(r); }
  static __device__ __forceinline__ void store(bfu* p, const float* y) { *p = f2bf(y[0]); }
};
template <>
struct Px<bfu, 2> {
  unsigned r;
  __device__ __forceinline__ void load(const bfu* p) { r = *(const unsigned*)p; }
  __device__ __forceinline__ float get(int i) const { return __builtin_bit_cast(float, i ? r & 0xffff0000u : r << 16); }
  static __device__ __forceinline__ void store(bfu* p, const float* y) { *(unsigned*)p = (unsigned)f2bf(y[0]) | (unsigned)f2bf(y[1]) << 16; }
};

template <typename T, int VEC, int CM, int KM, int MODE>
__global__ void __launch_bounds__(256) k_distill_planes(const DistP a) {
  using E = El<T>;
  using P = Px<T, VEC>;
  constexpr int BL = 8;
  const long long first = ((long long)blockIdx.x * 256 + threadIdx.x) * VEC;
  const bool in = first < a.N;
  float total = 0.f;
  if (in) {
    const T* z = (const T*)a.z + first;
    T* dz = (T*)a.dz + first;
    P x[CM > 0 ? CM : BL];
    float m[VEC], l[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) m[v] = -INFINITY, l[v] = 0.f;
    if constexpr (CM > 0) {
#pragma unroll
      for (int c = 0; c < CM; ++c)
        if (c < a.C) x[c].load(z + c * a.z_cs);
    }
    // the teacher's entries of the lane's rows
    int cl[KM > 0 ? KM * VEC : 1];
    float tl[KM > 0 ? KM * VEC : 1], zl[KM > 0 ? KM * VEC : 1];
    if constexpr (KM > 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
#pragma unroll
        for (int k = 0; k < KM; ++k)
          if (k < a.K) cl[v * KM + k] = entry_class(a, first + v, k), tl[v * KM + k] = entry_logit(a, first + v, k);
          else cl[v * KM + k] = -1;
#pragma unroll
      for (int v = 0; v < VEC; ++v)
#pragma unroll
        for (int k = 0; k < KM; ++k) {
          const int c = cl[v * KM + k];
          zl[v * KM + k] = c >= 0 ? E::load(z + v + c * a.z_cs) : 0.f;
        }
    }
    float l2[VEC];
    bool walk = MODE != BWD;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      l2[v] = MODE == BWD ? a.lse_in[first + v] * LOG2E : 0.f;
      walk |= MODE == BWD && !lse_serves(l2[v]);
    }
    if (walk) {
      if constexpr (CM > 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
          for (int c = 0; c < CM; ++c)
            if (c < a.C) m[v] = fmaxf(m[v], x[c].get(v));
          const float b = base_of(m[v]);
#pragma unroll
          for (int c = 0; c < CM; ++c)
            if (c < a.C) l[v] += exp2_((x[c].get(v) - b) * a.c);
        }
      } else {
        for (int c0 = 0; c0 < a.C; c0 += BL) {
#pragma unroll
          for (int c = 0; c < BL; ++c) x[c].load(z + min(c0 + c, a.C - 1) * a.z_cs);
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            float mx = m[v];
#pragma unroll
            for (int c = 0; c < BL; ++c) mx = fmaxf(mx, x[c].get(v));
            const float b = base_of(mx);
            l[v] *= exp2_((m[v] - b) * a.c);
            m[v] = mx;
#pragma unroll
            for (int c = 0; c < BL; ++c) l[v] += c0 + c < a.C ? exp2_((x[c].get(v) - b) * a.c) : 0.f;
          }
        }
      }
    }
    float mt[VEC], lt2[VEC], f[VEC], fi[VEC];
    bool empty[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const long long row = first + v;
      const auto entry = [&](int k) { return KM > 0 ? cl[v * KM + k] : entry_class(a, row, k); };
      const auto logit = [&](int k) { return KM > 0 ? tl[v * KM + k] : entry_logit(a, row, k); };
      mt[v] = -INFINITY;
      float lt = 0.f;
      if constexpr (KM > 0) {
#pragma unroll
        for (int k = 0; k < KM; ++k)
          if (entry(k) >= 0) mt[v] = fmaxf(mt[v], logit(k));
        const float b = base_of(mt[v]);
#pragma unroll
        for (int k = 0; k < KM; ++k)
          if (entry(k) >= 0) lt += exp2_((logit(k) - b) * a.c);
      } else {
        for (int k = 0; k < a.K; ++k)
          if (entry(k) >= 0) merge(mt[v], lt, logit(k), 1.f, a.c);
      }
      const float wt = a.w ? a.w[row] : 1.f;
      empty[v] = wt == 0.f || (!(lt > 0.f) && lt == lt);  // left out, or no entry at all
      lt2[v] = log2_(lt);
      if (MODE == BWD && lse_serves(l2[v])) m[v] = 0.f;
      else l2[v] = log2_(l[v]);
      if (MODE != BWD) {
        float loss = 0.f;
        const auto add = [&](int k) {
          const int c = entry(k);
          if (c < 0) return;
          const float lp = (logit(k) - mt[v]) * a.c - lt2[v], p = exp2_(lp);
          const float zc = KM > 0 ? zl[v * KM + k] : E::load(z + v + c * a.z_cs);
          if (!(p == 0.f)) loss += p * (lp - ((zc - m[v]) * a.c - l2[v]));
        };
        if constexpr (KM > 0) {
#pragma unroll
          for (int k = 0; k < KM; ++k) add(k);
        } else {
          for (int k = 0; k < a.K; ++k) add(k);
        }
        loss = empty[v] ? 0.f : loss * LN2 * a.T * a.T * wt;
        if (a.loss_each) a.loss_rows[row] = loss;
        total += loss;
        if (MODE == FWD) a.lse[row] = row_lse(a, m[v], l2[v]);
      }
      if (MODE != FWD) f[v] = row_factor(a, row, wt), fi[v] = MODE == BWD ? 0.f : f[v] * (1.f / l[v]);
    }
    if (MODE != FWD) {
      const auto grad = [&](float x, int v) {
        const float u = (x - m[v]) * a.c;
        return MODE == BWD ? f[v] * exp2_(u - l2[v]) : fi[v] * exp2_(u);
      };
      if constexpr (CM > 0) {
#pragma unroll
        for (int c = 0; c < CM; ++c)
          if (c < a.C) {
            float y[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) y[v] = empty[v] ? 0.f : grad(x[c].get(v), v);
            P::store(dz + c * a.d_cs, y);
          }
      } else {
        for (int c0 = 0; c0 < a.C; c0 += BL) {
#pragma unroll
          for (int c = 0; c < BL; ++c) x[c].load(z + min(c0 + c, a.C - 1) * a.z_cs);
#pragma unroll
          for (int c = 0; c < BL; ++c)
            if (c0 + c < a.C) {
              float y[VEC];
#pragma unroll
              for (int v = 0; v < VEC; ++v) y[v] = empty[v] ? 0.f : grad(x[c].get(v), v);
              P::store(dz + (c0 + c) * a.d_cs, y);
            }
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {  // the teacher's classes again, by the lane that wrote them; a class that stands there
        if (empty[v]) continue;        // twice has both probabilities in its sum
        const long long row = first + v;
        if constexpr (KM > 0) {
          float pk[KM];
#pragma unroll
          for (int k = 0; k < KM; ++k) pk[k] = cl[v * KM + k] >= 0 ? exp2_((tl[v * KM + k] - mt[v]) * a.c - lt2[v]) : 0.f;
#pragma unroll
          for (int k = 0; k < KM; ++k) {
            const int c = cl[v * KM + k];
            float p = 0.f;
#pragma unroll
            for (int j = 0; j < KM; ++j) p += cl[v * KM + j] == c ? pk[j] : 0.f;
            if (c >= 0) E::store(dz + v + c * a.d_cs, grad(zl[v * KM + k], v) - f[v] * p);
          }
        } else {
          for (int k = 0; k < a.K; ++k) {
            const int c = entry_class(a, row, k);
            if (c < 0) continue;
            float p = 0.f;
            for (int j = 0; j < a.K; ++j)
              if (entry_class(a, row, j) == c) p += exp2_((entry_logit(a, row, j) - mt[v]) * a.c - lt2[v]);
            E::store(dz + v + c * a.d_cs, grad(E::load(z + v + c * a.z_cs), v) - f[v] * p);
          }
        }
      }
    }
  }
  if (MODE != BWD && !a.loss_each) {  // one sum per workgroup
    __shared__ float part[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x == 0) a.loss_rows[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
  }
}

// Sum of n losses (of rows, or of workgroups of planes) by one workgroup, in 64 bits; eight of a thread's loads in flight.
__global__ void __launch_bounds__(1024) k_distill_sum(const float* __restrict__ x, long long n, float scale, float* __restrict__ out) {
  __shared__ double part[16];
  double s = 0.;
  for (long long i = threadIdx.x; i < n; i += 8192) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = i + 1024 * j < n ? x[i + 1024 * j] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)y[j];
  }
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
  // Threads by the length of the row: a wave where that gives each lane at most 4 chunks, then workgroups whose registers hold
  // the row while as many others as possible share the CU (their loads run under this one's arithmetic).
  const int nch = a.C / El<T>::EP;  // whole chunks at most
  const dim3 grid((unsigned)a.N);
#define GPN_ROWS(NT, CH, MANY) hipLaunchKernelGGL((k_distill_rows<T, NT, CH, MANY, MODE>), grid, dim3(NT), 0, st, a)
  if (nch <= 64) GPN_ROWS(64, 1, false);
  else if (nch <= 256) GPN_ROWS(64, 4, false);
  else if (nch <= 1024) GPN_ROWS(256, 4, false);
  else if (nch <= 2048) GPN_ROWS(256, 8, false);
  else if (nch <= 4096) GPN_ROWS(512, 8, false);
  else if (nch <= 8192) GPN_ROWS(512, 16, false);
  else if (nch <= 16384) GPN_ROWS(1024, 16, false);
  else GPN_ROWS(1024, 8, true);
#undef GPN_ROWS
}

template <typename T, int VEC, int MODE>
void launch_planes(const DistP& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.N + 256 * VEC - 1) / (256 * VEC)));
#define GPN_PLANES(CM, KM) hipLaunchKernelGGL((k_distill_planes<T, VEC, CM, KM, MODE>), grid, dim3(256), 0, st, a)
  if (a.C <= 32) {
    if (a.K <= 8) GPN_PLANES(32, 8);
    else GPN_PLANES(32, 0);
  } else {
    if (a.K <= 8) GPN_PLANES(0, 8);
    else GPN_PLANES(0, 0);
  }
#undef GPN_PLANES
}

template <int MODE>
int run(const gpn_distill_args_t* x, hipStream_t st, const char* name) {
  GPN_REQUIRE(x, "%s: null arguments", name);
  GPN_REQUIRE(x->dtype == GPN_DT_F32 || x->dtype == GPN_DT_BF16, "%s: unknown dtype %d", name, x->dtype);
  GPN_REQUIRE(x->teacher_dtype == GPN_DT_F32 || x->teacher_dtype == GPN_DT_BF16, "%s: unknown teacher dtype %d", name, x->teacher_dtype);
  GPN_REQUIRE(x->index_bytes == 4 || x->index_bytes == 8, "%s: indices of %d bytes", name, x->index_bytes);
  GPN_REQUIRE(x->N >= 0 && x->N <= INT_MAX, "%s: %lld rows", name, x->N);
  GPN_REQUIRE(x->C >= 1 && x->C <= (1 << 29), "%s: %d classes", name, x->C);
  GPN_REQUIRE(x->K >= 0 && x->K <= GPN_DISTILL_MAX_K, "%s: K must be in [0,%d] (got %d)", name, GPN_DISTILL_MAX_K, x->K);
  // its square and its reciprocal stay far within fp32
  GPN_REQUIRE(x->temperature >= 1e-12f && x->temperature <= 1e12f, "%s: temperature must be between 1e-12 and 1e12", name);
  GPN_REQUIRE(x->reduction >= GPN_RED_NONE && x->reduction <= GPN_RED_MEAN, "%s: unknown reduction %d", name, x->reduction);
  GPN_REQUIRE(x->logits || x->N == 0, "%s: null logits", name);
  GPN_REQUIRE((x->teacher && x->index) || x->K == 0 || x->N == 0, "%s: null teacher", name);
  const bool planes = x->class_stride != 1 && x->C > 1;
  GPN_REQUIRE(!planes || x->row_stride == 1 || x->N <= 1, "%s: logits need contiguous classes or contiguous rows (strides %lld, %lld)",
              name, x->row_stride, x->class_stride);
  GPN_REQUIRE(planes || x->N <= GPN_DISTILL_MAX_ROWS, "%s: %lld rows of contiguous classes", name, x->N);
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
  a.loss_each = x->reduction == GPN_RED_NONE;
  long long losses = x->N;  // values in loss_rows that make up the loss
  if (x->N > 0) {
    // bf16 planes: two rows per lane where every plane starts on 4 bytes
    const bool pairs = x->N % 2 == 0 && x->class_stride % 2 == 0 && x->dclass_stride % 2 == 0 &&
                       (((size_t)x->logits | (size_t)x->dlogits) & 3) == 0;
    if (planes) losses = (x->N + 255) / 256;
    if (planes && x->dtype == GPN_DT_F32) launch_planes<float, 1, MODE>(a, st);
    else if (planes && pairs) losses = (x->N + 511) / 512, launch_planes<bfu, 2, MODE>(a, st);
    else if (planes) launch_planes<bfu, 1, MODE>(a, st);
    else if (x->dtype == GPN_DT_F32) launch_rows<float, MODE>(a, st);
    else launch_rows<bfu, MODE>(a, st);
    GPN_LAUNCH_CHECK(name);
  }
  if (MODE != BWD && x->reduction != GPN_RED_NONE) {
    hipLaunchKernelGGL(k_distill_sum, dim3(1), dim3(1024), 0, st, x->loss_rows, losses, mean, x->loss);
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
