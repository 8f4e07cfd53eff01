// Softmax attention with its backward pass (gpn_attn_forward, gpn_attn_backward) for gfx950.
//
// One key/value head with the query heads that share it is one problem: its ROWS are the pairs (query position i, member
// g of the group), row = i * G + g, so shared heads read their keys once and the gradients of keys and values sum over the
// group inside a workgroup.
//
// Every product runs on MFMA in one orientation: the STATIONARY side (queries, in the forward and dq kernels; keys, in the
// dk / dv kernel) sits on the lanes (the n index of a tile), the side that is walked comes from LDS as the m index.
//   scores        S^T = K Q^T        A = rows of K (LDS, contiguous along d), B = rows of Q (registers)
//   outputs       O^T = V^T P^T      A = columns of V (LDS, read transposed),  B = P^T: the very registers S^T left
// The accumulator of a tile holds, per lane, one column and the rows crow(r, h); the B operand wants the rows 8h.. (bf16)
// or one row per lane group (fp32).  A sum over rows may take them in any order, so the A side is read in the order that
// the accumulator has: P never leaves the registers.  A row's softmax is then over registers of one lane and one (bf16) or
// two (fp32) exchanges between the lanes that share a column.
#include <climits>
#include <type_traits>

#include "common.h"

typedef __bf16 bf16;
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef float fl4 __attribute__((ext_vector_type(4)));
typedef float fl16 __attribute__((ext_vector_type(16)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ---------------------------------------------------------------------------------------------- matrix tiles per type
// TM: edge of a tile; NC: its accumulator registers per lane; EP: elements of a 16-byte fragment (16 steps of k over the
// lane groups); fragments of rows (rowfrag) are contiguous along d, fragments of columns (colfrag) run over 16 rows of the
// tile in the order crow() gives them.
template <typename T>
struct Mt;

template <>
struct Mt<bf16> {  // v_mfma_f32_32x32x16_bf16
  static constexpr int TM = 32, NC = 16, EP = 8;
  typedef bf8 Frag;
  typedef fl16 Acc;
  static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int crow(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }
  // fp32 -> bf16 (round to nearest even) of the 16 rows of group t: the probabilities and their gradients enter the second
  // product with 8 bits, which is what its other operand has; their sums stay fp32.
  static __device__ __forceinline__ Frag pack(const Acc& s, int t) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (bf16)s[8 * t + i];
    return f;
  }
  // ds_read_b64_tr_b16: lanes 4j .. 4j+3 of a group of 16 address 16 columns of row j; lane l receives column l of the four.
  static __device__ __forceinline__ Frag colfrag(const bf16* x, int ld, int lane) {
    const bf16* p = x + (4 * (lane >> 5) + ((lane & 15) >> 2)) * ld + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    typedef __attribute__((address_space(3))) s4v* lp;
    const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p);
    const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 8 * ld));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

template <>
struct Mt<float> {  // v_mfma_f32_16x16x4_f32, four of them per fragment
  static constexpr int TM = 16, NC = 4, EP = 4;
  typedef fl4 Frag;
  typedef fl4 Acc;
  static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ int crow(int r, int h) { return 4 * h + r; }
  static __device__ __forceinline__ Frag pack(const Acc& s, int) { return s; }
  static __device__ __forceinline__ Frag colfrag(const float* x, int ld, int lane) {
    const float* p = x + 4 * (lane >> 4) * ld + (lane & 15);
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = p[i * ld];
    return f;
  }
};

template <typename T>
__device__ __forceinline__ typename Mt<T>::Frag rowfrag(const T* x, int ld, int lane) {
  using M = Mt<T>;
  return *(const typename M::Frag*)(x + (lane & (M::TM - 1)) * ld + M::EP * (lane / M::TM));
}

// Combination over the lane groups that share a column (lanes n, n + TM, ..).  The values come from vector instructions, not
// from MFMA results in flight; s_nop 1 covers the distance v_permlane*_swap wants from them.
__device__ __forceinline__ void swap16(float v, float& a, float& b) {
  a = v, b = v;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void swap32(float v, float& a, float& b) {
  a = v, b = v;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
template <typename T>
__device__ __forceinline__ float col_max(float v) {
  float a, b;
  if (Mt<T>::TM == 16) {
    swap16(v, a, b);
    v = fmaxf(a, b);
  }
  swap32(v, a, b);
  return fmaxf(a, b);
}
template <typename T>
__device__ __forceinline__ float col_sum(float v) {
  float a, b;
  if (Mt<T>::TM == 16) {
    swap16(v, a, b);
    v = a + b;
  }
  swap32(v, a, b);
  return a + b;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

// Row strides of the LDS tiles (elements).  Rows read along d: 16 bytes more than a multiple of 64 banks spreads 16 rows over
// all of them.  bf16 columns (transposed reads touch 4 rows x 64 bytes at a time): 16 banks between rows.
template <typename T, int DP>
struct Ld {
  static constexpr int DV = (sizeof(T) == 2 && DP < 32) ? 32 : DP;  // columns that whole tiles of the output product cover
  static constexpr int row = DP + 16 / sizeof(T);
  static constexpr int col = sizeof(T) == 4 ? DP + 4 : (DV % 128 == 0 ? DV + 32 : DV % 64 == 0 ? DV + 32 : DV);
  static constexpr int both = DV + 16 / sizeof(T);
};

struct Strides {
  long long b, l, h;
};

struct AttnP {
  const void *q, *k, *v, *dout;
  void *out, *dq, *dk, *dv;
  Strides sq, sk, sv, sdo;
  float *lse, *delta, *part_o, *part_l;
  const int *lengths, *q_start;
  const unsigned char* key_mask;
  long long mask_sb;
  int B, Lq, Lk, Hq, Hkv, D, G, M;  // M = Lq * G rows of a problem
  unsigned g_magic;                 // row / G = umulhi(row, g_magic) for G > 1 (rows <= 2^24, G <= 256)
  int causal, tiles, nsplit, split_keys;
  float c;      // scale * log2(e)
  float scale;
};

__device__ __forceinline__ int row_pos(const AttnP& a, int row) { return a.G == 1 ? row : (int)__umulhi((unsigned)row, a.g_magic); }

// Workgroup -> (problem, unit of the problem).  Workgroups go to the eight XCDs in turn: problems are taken in groups of
// eight, so that all units of a problem meet in one L2, and units of one problem follow each other.  With one unit per
// problem each XCD takes a run of neighbouring problems instead: heads of a position share 128-byte lines.
__device__ __forceinline__ bool locate(int nprob, int units, int& p, int& u) {
  const int bid = blockIdx.x;
  if (units == 1) {
    const int per = (nprob + 7) >> 3;
    p = (bid & 7) * per + (bid >> 3), u = 0;
    return (bid >> 3) < per && p < nprob;
  }
  const int grp = bid / (8 * units), in = bid - grp * 8 * units, n = min(8, nprob - grp * 8);
  p = grp * 8 + in % n, u = in / n;
  return true;
}
inline long long grid_of(long long nprob, long long units) { return units == 1 ? (nprob + 7) / 8 * 8 : nprob * units; }

struct Prob {
  int b, hk, len, qs;
};
__device__ __forceinline__ Prob problem(const AttnP& a, int p) {
  Prob r;
  r.b = p / a.Hkv, r.hk = p - r.b * a.Hkv;
  r.len = a.lengths ? min(max(a.lengths[r.b], 0), a.Lk) : a.Lk;
  // a start beyond the keys (or before them by more than the queries) says no more than one at that distance
  r.qs = a.q_start ? min(max(a.q_start[r.b], -a.Lq), a.Lk) : a.Lk - a.Lq;
  return r;
}

// ROWS rows of DP elements, staged through registers: load() requests them, store() writes them to LDS.  Rows that `ok`
// refuses are zero and never read: hidden keys may hold anything.
template <typename T, int DP, int ROWS, int NTH>
struct Stage {
  static constexpr int EP = Mt<T>::EP, CPR = DP / EP, N = ROWS * CPR, NCH = (N + NTH - 1) / NTH;
  u4v r[NCH];
  template <typename RowPtr>
  __device__ __forceinline__ void load(int D, RowPtr row) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = threadIdx.x + i * NTH, j = c / CPR, e = (c % CPR) * EP;
      r[i] = u4v{0, 0, 0, 0};
      if ((N % NTH == 0 || c < N) && e < D) {
        const T* p = row(j);
        if (p) r[i] = *(const u4v*)(p + e);
      }
    }
  }
  __device__ __forceinline__ void store(T* lds, int ld) const {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = threadIdx.x + i * NTH;
      if (N % NTH == 0 || c < N) *(u4v*)(lds + (c / CPR) * ld + (c % CPR) * EP) = r[i];
    }
  }
};

// fragments of the stationary rows, straight from global memory (zero where p is null or d >= D)
template <typename T, int KF>
__device__ __forceinline__ void load_frags(typename Mt<T>::Frag (&f)[KF], const T* p, int D, int h) {
#pragma unroll
  for (int i = 0; i < KF; ++i) {
    const int d = 16 * i + Mt<T>::EP * h;
    u4v x = {0, 0, 0, 0};
    if (p && d < D) x = *(const u4v*)(p + d);
    f[i] = __builtin_bit_cast(typename Mt<T>::Frag, x);
  }
}

// one column (lane n) of an accumulator over DP rows, times f -> row at p
template <typename T, typename TO, int MD>
__device__ __forceinline__ void store_cols(const typename Mt<T>::Acc (&o)[MD], float f, TO* p, int D, int h) {
  using M = Mt<T>;
#pragma unroll
  for (int md = 0; md < MD; ++md)
#pragma unroll
    for (int q = 0; q < M::NC / 4; ++q) {
      const int d = md * M::TM + M::crow(4 * q, h);
      if (d < D) {
        typedef TO V4 __attribute__((ext_vector_type(4)));
        V4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (TO)(o[md][4 * q + i] * f);
        *(V4*)(p + d) = x;
      }
    }
}

// ---------------------------------------------------------------------------------------------------- forward
// WM waves along the rows x WK waves along the keys; a wave walks KT keys of every stage of WK * KT.
template <typename T, int DP, int WM, int WK, int KT, int NBUF>
struct Fwd {
  using M = Mt<T>;
  static constexpr int TM = M::TM, MT = KT / TM, BN = WK * KT, BM = WM * TM, NTH = 64 * WM * WK, KF = DP / 16;
  static constexpr int DV = Ld<T, DP>::DV, MD = DV / TM, LK = Ld<T, DP>::row, LV = Ld<T, DP>::col, LO = DV + 4;
  static constexpr size_t stage_bytes = (size_t)NBUF * BN * (LK + LV) * sizeof(T);
  static constexpr size_t join_bytes = WK > 1 ? (size_t)WK * BM * (LO + 2) * 4 : 0;
  static constexpr size_t lds = stage_bytes > join_bytes ? stage_bytes : join_bytes;
};

extern __shared__ __attribute__((aligned(16))) unsigned char attn_smem[];

template <typename T, int DP, int WM, int WK, int KT, int NBUF>
__global__ void __launch_bounds__(64 * WM * WK, 2) k_attn_fwd(const AttnP a) {
  using F = Fwd<T, DP, WM, WK, KT, NBUF>;
  using M = Mt<T>;
  constexpr int TM = F::TM, MT = F::MT, BN = F::BN, BM = F::BM, NTH = F::NTH, KF = F::KF, MD = F::MD, LK = F::LK, LV = F::LV;
  int pr, unit;
  if (!locate(a.B * a.Hkv, a.tiles * a.nsplit, pr, unit)) return;
  const int split = unit / a.tiles, tile = a.tiles - 1 - (unit - split * a.tiles);  // causal: the longest tiles first
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wk = wave % WK, wm = wave / WK;
  const int n = lane & (TM - 1), h = lane / TM;
  const int row = tile * BM + wm * TM + n;
  const bool live = row < a.M;
  const int i = row_pos(a, live ? row : 0), g = (live ? row : 0) - i * a.G, hq = p.hk * a.G + g;
  const int lim = a.causal ? p.qs + i : INT_MAX;  // last key this row may see

  int kend = p.len;
  if (a.causal) kend = min(kend, p.qs + row_pos(a, min(tile * BM + BM, a.M) - 1) + 1);
  int kbeg = 0;
  if (a.nsplit > 1) kbeg = split * a.split_keys, kend = min(kend, kbeg + a.split_keys);

  typename M::Frag qf[KF];
  load_frags<T, KF>(qf, live ? (const T*)a.q + p.b * a.sq.b + i * a.sq.l + hq * a.sq.h : nullptr, a.D, h);

  const T* kb = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* vb = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const unsigned char* km = a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr;
  T* ks = (T*)attn_smem;
  T* vs = ks + NBUF * BN * LK;
  Stage<T, DP, BN, NTH> sk, sv;
  const auto request = [&](int j0) {
    sk.load(a.D, [&](int j) { return j0 + j < kend && (!km || km[j0 + j]) ? kb + (j0 + j) * a.sk.l : (const T*)nullptr; });
    sv.load(a.D, [&](int j) { return j0 + j < kend && (!km || km[j0 + j]) ? vb + (j0 + j) * a.sv.l : (const T*)nullptr; });
  };
  const int stages = kend > kbeg ? (kend - kbeg + BN - 1) / BN : 0;

  typename M::Acc o[MD];
#pragma unroll
  for (int md = 0; md < MD; ++md) o[md] = (typename M::Acc)(0.f);
  float m = -INFINITY, l = 0.f;  // running maximum of the raw scores; this lane's share of the sum

  if (stages) {
    request(kbeg);
    if (NBUF == 2) {
      sk.store(ks, LK), sv.store(vs, LV);
      if (stages > 1) request(kbeg + BN);
      __syncthreads();
    }
  }
  for (int s = 0; s < stages; ++s) {
    const int j0 = kbeg + s * BN;
    if (NBUF == 2) {
      if (s + 1 < stages) {
        sk.store(ks + ((s + 1) & 1) * BN * LK, LK), sv.store(vs + ((s + 1) & 1) * BN * LV, LV);
        if (s + 2 < stages) request(j0 + 2 * BN);
      }
    } else {
      sk.store(ks, LK), sv.store(vs, LV);
      __syncthreads();
      if (s + 1 < stages) request(j0 + BN);
    }
    const T* kt = ks + (NBUF == 2 ? (s & 1) * BN * LK : 0) + wk * KT * LK;
    const T* vt = vs + (NBUF == 2 ? (s & 1) * BN * LV : 0) + wk * KT * LV;
    const int jw = j0 + wk * KT;
    const bool key_ok = lane < KT && jw + lane < kend && (!km || km[jw + lane]);
    unsigned long long bits = __ballot(key_ok);
    if (bits && !__all(lim < jw)) {
      typename M::Acc sc[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sc[mt] = (typename M::Acc)(0.f);
#pragma unroll
        for (int f = 0; f < KF; ++f) sc[mt] = M::mma(rowfrag<T>(kt + mt * TM * LK + 16 * f, LK, lane), qf[f], sc[mt]);
      }
      constexpr unsigned long long ALL = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
      if (bits != ALL || __any(lim < jw + KT - 1)) {
        // bit x of the lane: key jw + x is visible to its row
        if (lim < jw + KT - 1) bits &= lim < jw ? 0ull : ~0ull >> (63 - (lim - jw));
        bits >>= 4 * h;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < M::NC; ++r)
            if (!(bits >> (mt * TM + M::crow(r, 0)) & 1)) sc[mt][r] = -INFINITY;
      }
      float mx = sc[0][0];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < M::NC; ++r) mx = fmaxf(mx, sc[mt][r]);
      // The row's reference moves only when a score exceeds it by 8 powers of two: until then the sums just grow, in fp32, and
      // the products' operands keep their relative precision.  alpha is 1 for the rows of the wave that stay.
      mx = col_max<T>(mx);
      const bool grow = (mx - m) * a.c > 8.f;  // of a row without a key so far: inf > 8; still without: nan > 8
      if (__any(grow)) {
        const float alpha = grow ? exp2_((m - mx) * a.c) : 1.f;
        m = grow ? mx : m;
        l *= alpha;
#pragma unroll
        for (int md = 0; md < MD; ++md) o[md] *= alpha;
      }
      const float mc = m == -INFINITY ? 0.f : m * a.c;
      float sum = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < M::NC; ++r) {
          const float e = exp2_(__builtin_fmaf(sc[mt][r], a.c, -mc));
          sc[mt][r] = e;
          sum += e;
        }
      l += sum;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < TM / 16; ++t) {
          const typename M::Frag pf = M::pack(sc[mt], t);
#pragma unroll
          for (int md = 0; md < MD; ++md)
            o[md] = M::mma(M::colfrag(vt + (mt * TM + 16 * t) * LV + md * TM, LV, lane), pf, o[md]);
        }
    }
    __syncthreads();
  }
  l = col_sum<T>(l);

  if (WK > 1) {  // join the waves that walked different keys
    constexpr int LO = F::LO;
    float* mo = (float*)attn_smem;  // [WK][BM] maxima, [WK][BM] sums, [WK][BM][LO] outputs
    float* lo = mo + WK * BM;
    float* oo = lo + WK * BM;
    // every wave is past its last read of the stages (the barrier that ends the loop; without a stage nothing was read)
    if (h == 0) mo[wk * BM + wm * TM + n] = m, lo[wk * BM + wm * TM + n] = l;
#pragma unroll
    for (int md = 0; md < MD; ++md)
#pragma unroll
      for (int q = 0; q < M::NC / 4; ++q) {
        fl4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = o[md][4 * q + e];
        *(fl4*)(oo + (wk * BM + wm * TM + n) * LO + md * TM + M::crow(4 * q, h)) = x;
      }
    __syncthreads();
    for (int x = threadIdx.x; x < BM * (DP / 4); x += NTH) {
      const int rr = x / (DP / 4), d = 4 * (x % (DP / 4)), rw = tile * BM + rr;
      if (rw >= a.M) continue;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < WK; ++w) mm = fmaxf(mm, mo[w * BM + rr]);
      const float ms = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      fl4 acc = (fl4)(0.f);
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float f = exp2_((mo[w * BM + rr] - ms) * a.c);
        ll += f * lo[w * BM + rr];
        acc += f * *(const fl4*)(oo + (w * BM + rr) * LO + d);
      }
      acc *= ll > 0.f || ll != ll ? 1.f / ll : 0.f;
      const float l2 = ll == 0.f ? -INFINITY : ms * a.c + log2_(ll);
      const int ii = row_pos(a, rw), hh = p.hk * a.G + rw - ii * a.G;
      if (a.nsplit > 1) {
        const long long at = ((long long)split * a.B * a.Hkv + pr) * a.M + rw;
        if (d == 0) a.part_l[at] = l2;
        if (d < a.D) *(fl4*)(a.part_o + at * a.D + d) = acc;
      } else {
        if (d == 0) a.lse[((long long)p.b * a.Hq + hh) * a.Lq + ii] = l2 * LN2;
        typedef T V4 __attribute__((ext_vector_type(4)));
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)acc[e];
        if (d < a.D) *(V4*)((T*)a.out + (((long long)p.b * a.Lq + ii) * a.Hq + hh) * a.D + d) = y;
      }
    }
    return;
  }
  if (!live) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row without a key is zero
  const float l2 = l == 0.f ? -INFINITY : m * a.c + log2_(l);
  if (a.nsplit > 1) {
    const long long at = ((long long)split * a.B * a.Hkv + pr) * a.M + row;
    if (h == 0) a.part_l[at] = l2;
    store_cols<T, float, MD>(o, inv, a.part_o + at * a.D, a.D, h);
    return;
  }
  if (h == 0) a.lse[((long long)p.b * a.Hq + hq) * a.Lq + i] = l2 * LN2;
  store_cols<T, T, MD>(o, inv, (T*)a.out + (((long long)p.b * a.Lq + i) * a.Hq + hq) * a.D, a.D, h);
}

// Joins the splits of a row: every split left its own normalised output and log2-sum-exp.  32 lanes per row, 4 values a lane.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_join(const AttnP a) {
  const long long x = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (long long)a.B * a.Hkv * a.M;
  const int d = 4 * (threadIdx.x & 31);
  if (x >= rows) return;
  const int pr = (int)(x / a.M), row = (int)(x - (long long)pr * a.M);
  const int b = pr / a.Hkv, i = row_pos(a, row), hq = (pr - b * a.Hkv) * a.G + row - i * a.G;
  float mm = -INFINITY;
  bool bad = false;
  for (int s = 0; s < a.nsplit; ++s) {
    const float l2 = a.part_l[s * rows + x];
    mm = fmaxf(mm, l2), bad |= l2 != l2;
  }
  const float ms = mm == -INFINITY ? 0.f : mm;
  float w = 0.f;
  fl4 acc = (fl4)(0.f);
  for (int s = 0; s < a.nsplit; ++s) {
    const float f = exp2_(a.part_l[s * rows + x] - ms);
    w += f;
    if (d < a.D) acc += f * *(const fl4*)(a.part_o + (s * rows + x) * a.D + d);
  }
  acc *= w > 0.f || bad ? 1.f / w : 0.f;
  if (d == 0) a.lse[((long long)b * a.Hq + hq) * a.Lq + i] = w == 0.f ? -INFINITY : (ms + log2_(w)) * LN2;
  typedef T V4 __attribute__((ext_vector_type(4)));
  V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)acc[e];
  if (d < a.D) *(V4*)((T*)a.out + (((long long)b * a.Lq + i) * a.Hq + hq) * a.D + d) = y;
}

// ---------------------------------------------------------------------------------------------------- gradient of queries
// Rows of queries and of the output's gradient are stationary; keys and values walk past.  The probabilities are computed
// again from the row's log-sum-exp, so a row's share of the work needs no maximum and no sum:
//   p = exp(s - lse), ds = p (do.v - delta), dq = scale sum ds k,  delta = do.o  (written out for the other kernel).
template <typename T, int DP, int WM, int KT>
struct Dq {
  using M = Mt<T>;
  static constexpr int TM = M::TM, MT = KT / TM, BM = WM * TM, NTH = 64 * WM, KF = DP / 16;
  static constexpr int DV = Ld<T, DP>::DV, MD = DV / TM, LK = Ld<T, DP>::both, LV = Ld<T, DP>::row;
  static constexpr size_t lds = (size_t)2 * KT * (LK + LV) * sizeof(T);
};

template <typename T, int DP, int WM, int KT>
__global__ void __launch_bounds__(64 * WM, 2) k_attn_dq(const AttnP a) {
  using F = Dq<T, DP, WM, KT>;
  using M = Mt<T>;
  constexpr int TM = F::TM, MT = F::MT, BM = F::BM, NTH = F::NTH, KF = F::KF, MD = F::MD, LK = F::LK, LV = F::LV;
  int pr, unit;
  if (!locate(a.B * a.Hkv, a.tiles, pr, unit)) return;
  const int tile = a.tiles - 1 - unit;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & (TM - 1), h = lane / TM;
  const int row = tile * BM + wave * TM + n;
  const bool live = row < a.M;
  const int i = row_pos(a, live ? row : 0), g = (live ? row : 0) - i * a.G, hq = p.hk * a.G + g;
  const int lim = a.causal ? p.qs + i : INT_MAX;
  int kend = p.len;
  if (a.causal) kend = min(kend, p.qs + row_pos(a, min(tile * BM + BM, a.M) - 1) + 1);

  typename M::Frag qf[KF], df[KF];
  load_frags<T, KF>(qf, live ? (const T*)a.q + p.b * a.sq.b + i * a.sq.l + hq * a.sq.h : nullptr, a.D, h);
  load_frags<T, KF>(df, live ? (const T*)a.dout + p.b * a.sdo.b + i * a.sdo.l + hq * a.sdo.h : nullptr, a.D, h);
  const long long at = ((long long)p.b * a.Hq + hq) * a.Lq + i, orow = (((long long)p.b * a.Lq + i) * a.Hq + hq) * a.D;
  float delta = 0.f;
  {
    typename M::Frag of[KF];
    load_frags<T, KF>(of, live ? (const T*)a.out + orow : nullptr, a.D, h);
#pragma unroll
    for (int f = 0; f < KF; ++f)
#pragma unroll
      for (int e = 0; e < M::EP; ++e) delta = __builtin_fmaf((float)df[f][e], (float)of[f][e], delta);
    delta = col_sum<T>(delta);
  }
  float lse2 = live ? a.lse[at] * LOG2E : INFINITY;
  if (lse2 == -INFINITY) lse2 = INFINITY;  // a row without a key: every probability is zero
  if (live && h == 0) a.delta[at] = delta;

  const T* kb = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* vb = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const unsigned char* km = a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr;
  T* ks = (T*)attn_smem;
  T* vs = ks + 2 * KT * LK;
  Stage<T, DP, KT, NTH> sk, sv;
  const auto request = [&](int j0) {
    sk.load(a.D, [&](int j) { return j0 + j < kend && (!km || km[j0 + j]) ? kb + (j0 + j) * a.sk.l : (const T*)nullptr; });
    sv.load(a.D, [&](int j) { return j0 + j < kend && (!km || km[j0 + j]) ? vb + (j0 + j) * a.sv.l : (const T*)nullptr; });
  };
  const int stages = kend > 0 ? (kend + KT - 1) / KT : 0;
  typename M::Acc dq[MD];
#pragma unroll
  for (int md = 0; md < MD; ++md) dq[md] = (typename M::Acc)(0.f);
  if (stages) {
    request(0);
    sk.store(ks, LK), sv.store(vs, LV);
    if (stages > 1) request(KT);
    __syncthreads();
  }
  for (int s = 0; s < stages; ++s) {
    const int j0 = s * KT;
    if (s + 1 < stages) {
      sk.store(ks + ((s + 1) & 1) * KT * LK, LK), sv.store(vs + ((s + 1) & 1) * KT * LV, LV);
      if (s + 2 < stages) request(j0 + 2 * KT);
    }
    const T* kt = ks + (s & 1) * KT * LK;
    const T* vt = vs + (s & 1) * KT * LV;
    unsigned long long bits = __ballot(lane < KT && j0 + lane < kend && (!km || km[j0 + lane]));
    if (bits && !__all(lim < j0)) {
      constexpr unsigned long long ALL = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
      const bool partly = bits != ALL || __any(lim < j0 + KT - 1);
      if (lim < j0 + KT - 1) bits &= lim < j0 ? 0ull : ~0ull >> (63 - (lim - j0));
      bits >>= 4 * h;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        typename M::Acc sc = (typename M::Acc)(0.f), dp = (typename M::Acc)(0.f);
#pragma unroll
        for (int f = 0; f < KF; ++f) {
          sc = M::mma(rowfrag<T>(kt + mt * TM * LK + 16 * f, LK, lane), qf[f], sc);
          dp = M::mma(rowfrag<T>(vt + mt * TM * LV + 16 * f, LV, lane), df[f], dp);
        }
#pragma unroll
        for (int r = 0; r < M::NC; ++r) {
          float e = exp2_(__builtin_fmaf(sc[r], a.c, -lse2));
          if (partly && !(bits >> (mt * TM + M::crow(r, 0)) & 1)) e = 0.f;
          sc[r] = e * (dp[r] - delta);
        }
#pragma unroll
        for (int t = 0; t < TM / 16; ++t) {
          const typename M::Frag sf = M::pack(sc, t);
#pragma unroll
          for (int md = 0; md < MD; ++md)
            dq[md] = M::mma(M::colfrag(kt + (mt * TM + 16 * t) * LK + md * TM, LK, lane), sf, dq[md]);
        }
      }
    }
    __syncthreads();
  }
  if (live) store_cols<T, T, MD>(dq, a.scale, (T*)a.dq + orow, a.D, h);
}

// ---------------------------------------------------------------------------------------------- gradients of keys, values
// Keys and values are stationary, a wave holds TM of them; the rows of all query heads that share them walk past, so the sum
// over the group is part of the walk and its order is fixed.  WN waves along the keys x WR waves along the rows: the WR waves of
// the same keys take the rows of a stage in turns and join their sums at the end, so that two waves fit a SIMD (256 registers)
// without a second copy of the keys' sums in memory.  Where those registers are short (VL) the values come from LDS.
// Work is cut evenly: under `causal` a workgroup takes the key tiles t and tiles - 1 - t, which together see as many rows as any
// other such pair, and every tile's own rows are cut into nsplit parts (fp32 sums in the workspace, joined in order).
template <typename T, int DP, int WN, int WR>
struct Dkv {
  using M = Mt<T>;
  static constexpr int TM = M::TM, RW = sizeof(T) == 4 && DP > 64 ? 16 : 32, RB = WR * RW, MT = RW / TM, BN = WN * TM, NTH = 64 * WN * WR, KF = DP / 16;
  static constexpr int DV = Ld<T, DP>::DV, MD = DV / TM, LQ = Ld<T, DP>::both, LV = Ld<T, DP>::row;
  static constexpr bool VL = DP > 64;
  static constexpr size_t stage_bytes = (size_t)2 * (2 * RB * LQ * sizeof(T) + 2 * RB * 4) + (VL ? BN * LV * sizeof(T) : 0);
  static constexpr size_t join_bytes = WR > 1 ? (size_t)WN * 2 * MD * M::NC * 64 * 4 : 0;
  static constexpr size_t lds = stage_bytes > join_bytes ? stage_bytes : join_bytes;
};

template <typename T, int DP, int WN, int WR>
__global__ void __launch_bounds__(64 * WN * WR, 2) k_attn_dkv(const AttnP a) {
  using F = Dkv<T, DP, WN, WR>;
  using M = Mt<T>;
  static_assert(WR == 1 || WR == 2, "the join below exchanges between two waves");
  constexpr int TM = F::TM, MT = F::MT, RB = F::RB, BN = F::BN, NTH = F::NTH, KF = F::KF, MD = F::MD, LQ = F::LQ, LV = F::LV;
  constexpr bool VL = F::VL;
  int pr, unit;
  if (!locate(a.B * a.Hkv, (a.causal ? (a.tiles + 1) / 2 : a.tiles) * a.nsplit, pr, unit)) return;
  const int tu = unit / a.nsplit, split = unit - tu * a.nsplit;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave % WN, wr = wave / WN;
  const int n = lane & (TM - 1), h = lane / TM;
  const unsigned char* km = a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr;
  const auto first_row = [&](int j) { return !a.causal || j <= p.qs ? 0 : j - p.qs >= a.Lq ? INT_MAX : (j - p.qs) * a.G; };

  T* qs = (T*)attn_smem;                   // [2][RB][LQ]
  T* ds = qs + 2 * RB * LQ;                // [2][RB][LQ]
  float* ls = (float*)(ds + 2 * RB * LQ);  // [2][RB] log-sum-exp (log2), [2][RB] delta
  T* vs = (T*)(ls + 4 * RB);               // [BN][LV]
  Stage<T, DP, RB, NTH> sq, sd;
  float rl, rd;
  const auto request = [&](int r0) {
    const auto at = [&](const void* base, const Strides& s, int r) -> const T* {
      r += r0;
      if (r >= a.M) return nullptr;
      const int i = row_pos(a, r);
      return (const T*)base + p.b * s.b + i * s.l + (p.hk * a.G + r - i * a.G) * s.h;
    };
    sq.load(a.D, [&](int r) { return at(a.q, a.sq, r); });
    sd.load(a.D, [&](int r) { return at(a.dout, a.sdo, r); });
    rl = INFINITY, rd = 0.f;
    const int r = r0 + threadIdx.x;
    if (threadIdx.x < RB && r < a.M) {
      const int i = row_pos(a, r);
      const long long x = ((long long)p.b * a.Hq + p.hk * a.G + r - i * a.G) * a.Lq + i;
      rl = a.lse[x] * LOG2E, rd = a.delta[x];
      if (rl == -INFINITY) rl = INFINITY;
    }
  };
  const auto put = [&](int buf) {
    sq.store(qs + buf * RB * LQ, LQ), sd.store(ds + buf * RB * LQ, LQ);
    if (threadIdx.x < RB) ls[buf * RB + threadIdx.x] = rl, ls[(2 + buf) * RB + threadIdx.x] = rd;
  };

  for (int half = 0; half < (a.causal ? 2 : 1); ++half) {
    const int tile = half ? a.tiles - 1 - tu : tu;
    if (half && tile <= tu) break;
    if (half) __syncthreads();  // the join of the first tile has been read
    const int j0 = tile * BN, key = j0 + wn * TM + n;
    const bool seen = key < p.len && (!km || km[key]);
    // first row that sees the lane's key / the wave's first key / all of the wave's keys
    const int rmin = first_row(key), rany = first_row(j0 + wn * TM), rall = first_row(j0 + wn * TM + TM - 1);
    int rbeg = j0 < p.len ? first_row(j0) : INT_MAX, rend = rbeg;
    if (rbeg < a.M) {
      const int b0 = rbeg / RB, blocks = (a.M + RB - 1) / RB - b0;
      rbeg = (b0 + (int)((long long)blocks * split / a.nsplit)) * RB;
      rend = min((b0 + (int)((long long)blocks * (split + 1) / a.nsplit)) * RB, a.M);
    }

    typename M::Frag kf[KF], vf[VL ? 1 : KF];
    load_frags<T, KF>(kf, seen ? (const T*)a.k + p.b * a.sk.b + key * a.sk.l + p.hk * a.sk.h : nullptr, a.D, h);
    if constexpr (VL) {
      Stage<T, DP, BN, NTH> sv;
      sv.load(a.D, [&](int j) {
        return j0 + j < p.len && (!km || km[j0 + j]) ? (const T*)a.v + p.b * a.sv.b + (j0 + j) * a.sv.l + p.hk * a.sv.h
                                                     : (const T*)nullptr;
      });
      sv.store(vs, LV);
    } else {
      load_frags<T, KF>(vf, seen ? (const T*)a.v + p.b * a.sv.b + key * a.sv.l + p.hk * a.sv.h : nullptr, a.D, h);
    }
    const T* vw = vs + wn * TM * LV;

    typename M::Acc dk[MD], dv[MD];
#pragma unroll
    for (int md = 0; md < MD; ++md) dk[md] = dv[md] = (typename M::Acc)(0.f);
    if (rbeg < rend) {
      request(rbeg);
      put(0);
      if (rbeg + RB < rend) request(rbeg + RB);
      __syncthreads();
    }
    int buf = 0;
    for (int r0 = rbeg; r0 < rend; r0 += RB, buf ^= 1) {
      if (r0 + RB < rend) {
        put(buf ^ 1);
        if (r0 + 2 * RB < rend) request(r0 + 2 * RB);
      }
      const int rw = r0 + wr * F::RW;
      if (rw + F::RW > rany) {
        const bool partly = rw < rall;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int lr = buf * RB + wr * F::RW + mt * TM;  // the tile's row in LDS
          const T* qt = qs + lr * LQ;
          const T* dt = ds + lr * LQ;
          typename M::Acc sc = (typename M::Acc)(0.f), dp = (typename M::Acc)(0.f);
#pragma unroll
          for (int f = 0; f < KF; ++f) {
            sc = M::mma(rowfrag<T>(qt + 16 * f, LQ, lane), kf[f], sc);
            if constexpr (VL) dp = M::mma(rowfrag<T>(dt + 16 * f, LQ, lane), rowfrag<T>(vw + 16 * f, LV, lane), dp);
            else dp = M::mma(rowfrag<T>(dt + 16 * f, LQ, lane), vf[f], dp);
          }
#pragma unroll
          for (int q = 0; q < M::NC / 4; ++q) {
            const int r = M::crow(4 * q, h);
            const fl4 l4 = *(const fl4*)(ls + lr + r), d4 = *(const fl4*)(ls + 2 * RB + lr + r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = exp2_(__builtin_fmaf(sc[4 * q + e], a.c, -l4[e]));
              if (partly && rw + mt * TM + r + e < rmin) x = 0.f;
              sc[4 * q + e] = x;
              dp[4 * q + e] = x * (dp[4 * q + e] - d4[e]);
            }
          }
#pragma unroll
          for (int t = 0; t < TM / 16; ++t) {
            const typename M::Frag pf = M::pack(sc, t), sf = M::pack(dp, t);
#pragma unroll
            for (int md = 0; md < MD; ++md) {
              dv[md] = M::mma(M::colfrag(dt + 16 * t * LQ + md * TM, LQ, lane), pf, dv[md]);
              dk[md] = M::mma(M::colfrag(qt + 16 * t * LQ + md * TM, LQ, lane), sf, dk[md]);
            }
          }
        }
      }
      __syncthreads();
    }
    if constexpr (WR == 2) {  // wave 0 of a pair finishes dk, wave 1 finishes dv
      fl4* x = (fl4*)attn_smem + (wn * 2) * MD * (M::NC / 4) * 64 + lane;
      const auto give = [&](const typename M::Acc(&o)[MD], int slot) {
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
          for (int q = 0; q < M::NC / 4; ++q) {
            fl4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = o[md][4 * q + e];
            x[((slot * MD + md) * (M::NC / 4) + q) * 64] = y;
          }
      };
      const auto take = [&](typename M::Acc(&o)[MD], int slot) {
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
          for (int q = 0; q < M::NC / 4; ++q) {
            const fl4 y = x[((slot * MD + md) * (M::NC / 4) + q) * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[md][4 * q + e] += y[e];
          }
      };
      if (rbeg >= rend) __syncthreads();  // no stage: the values' tile may still be on its way into the same memory
      if (wr) give(dk, 0);
      else give(dv, 1);
      __syncthreads();
      if (wr) take(dv, 1);
      else take(dk, 0);
    }
    if (key < a.Lk) {
      const long long at = (((long long)p.b * a.Lk + key) * a.Hkv + p.hk) * a.D;
      const long long part = (long long)a.B * a.Lk * a.Hkv * a.D;
      if (!seen) {  // a hidden key's gradients are zero, whatever stood in its row
#pragma unroll
        for (int md = 0; md < MD; ++md) dk[md] = dv[md] = (typename M::Acc)(0.f);
      }
      if (a.nsplit > 1) {
        if (WR == 1 || !wr) store_cols<T, float, MD>(dk, a.scale, a.part_o + 2 * split * part + at, a.D, h);
        if (WR == 1 || wr) store_cols<T, float, MD>(dv, 1.f, a.part_o + (2 * split + 1) * part + at, a.D, h);
      } else {
        if (WR == 1 || !wr) store_cols<T, T, MD>(dk, a.scale, (T*)a.dk + at, a.D, h);
        if (WR == 1 || wr) store_cols<T, T, MD>(dv, 1.f, (T*)a.dv + at, a.D, h);
      }
    }
  }
}

// Sums the parts of dk and dv in order.  4 values a lane.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_dkv_join(const AttnP a) {
  const long long part = (long long)a.B * a.Lk * a.Hkv * a.D;
  const long long x = 4 * ((long long)blockIdx.x * 256 + threadIdx.x);
  if (x >= 2 * part) return;
  fl4 s = (fl4)(0.f);
  for (int i = 0; i < a.nsplit; ++i) s += *(const fl4*)(a.part_o + 2 * i * part + x);
  typedef T V4 __attribute__((ext_vector_type(4)));
  V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)s[e];
  *(V4*)((T*)(x < part ? a.dk : a.dv) + (x < part ? x : x - part)) = y;
}

// ------------------------------------------------------------------------------------------------------------ host
template <typename K>
int launch(K kernel, const char* name, long long grid, int threads, size_t lds, hipStream_t st, const AttnP& a) {
  GPN_REQUIRE(grid <= INT_MAX, "%s: grid of %lld workgroups", name, grid);
  if (grid == 0) return GPN_OK;
  if (lds > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return gpn_set_error(GPN_E_LAUNCH, "hipFuncSetAttribute(%zu B LDS): %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, a);
  GPN_LAUNCH_CHECK(name);
  return GPN_OK;
}

// How a forward call is cut: rows per workgroup, keys per stage, splits of the keys.
struct Plan {
  bool few;  // few rows per problem: the waves of a workgroup share the rows and divide the keys
  int bm, tiles, nsplit, split_keys;
};

constexpr int MAX_SPLIT = 64;

Plan plan_forward(const gpn_attn_args_t* x) {
  Plan p;
  const bool f32 = x->dtype == GPN_DT_F32;
  const long long M = (long long)x->Lq * (x->Hq / x->Hkv), prob = (long long)x->B * x->Hkv;
  p.few = M <= (f32 ? 16 : 32);
  p.bm = p.few ? (f32 ? 16 : 32) : (f32 ? 64 : 128);
  p.tiles = (int)((M + p.bm - 1) / p.bm);
  const int bn = p.few ? 128 : 64;
  // Workgroups that find a CU of their own walk the keys alone; fewer than that, and the keys are cut, at 256 or more a
  // part so that a part outweighs its share of the join.
  const long long units = prob * p.tiles, want = 512;
  p.nsplit = 1, p.split_keys = x->Lk;
  if (units < want / 2 && x->Lk > 512) {
    long long s = want / units;
    if (s > MAX_SPLIT) s = MAX_SPLIT;
    const long long most = x->Lk / 256;
    if (s > most) s = most;
    if (s > 1) {
      p.split_keys = (int)(((x->Lk + s - 1) / s + bn - 1) / bn * bn);
      p.nsplit = (x->Lk + p.split_keys - 1) / p.split_keys;
    }
  }
  return p;
}

int check_args(const gpn_attn_args_t* x, const char* name) {
  GPN_REQUIRE(x, "%s: null arguments", name);
  GPN_REQUIRE(x->dtype == GPN_DT_F32 || x->dtype == GPN_DT_BF16, "%s: unknown dtype %d", name, x->dtype);
  GPN_REQUIRE(x->B >= 0 && x->Lq >= 0 && x->Lk >= 0, "%s: negative size", name);
  GPN_REQUIRE(x->Hq >= 1 && x->Hkv >= 1 && x->Hq % x->Hkv == 0, "%s: %d query heads cannot share %d key/value heads", name,
              x->Hq, x->Hkv);
  GPN_REQUIRE(x->D >= 8 && x->D <= GPN_ATTN_MAX_D && x->D % 8 == 0, "%s: head width must be a multiple of 8 up to %d (got %d)",
              name, GPN_ATTN_MAX_D, x->D);
  const int G = x->Hq / x->Hkv;
  GPN_REQUIRE(G <= 256 && (long long)x->Lq * G <= (1 << 24), "%s: %d queries x %d heads per key/value head", name, x->Lq, G);
  GPN_REQUIRE(x->Lk <= (1 << 30), "%s: %d keys", name, x->Lk);
  GPN_REQUIRE((long long)x->B * x->Hkv <= (1 << 24), "%s: %d batches x %d key/value heads", name, x->B, x->Hkv);
  GPN_REQUIRE(x->scale > 0.f && x->scale < INFINITY, "%s: scale must be positive and finite", name);
  return GPN_OK;
}

int check_tensor(const void* p, const long long* s, int size, const char* what, const char* name) {
  GPN_REQUIRE(p, "%s: null %s", name, what);
  GPN_REQUIRE(((size_t)p & 15) == 0, "%s: %s is not 16-byte aligned", name, what);
  for (int i = 0; s && i < 3; ++i)
    GPN_REQUIRE(s[i] >= 0 && s[i] * size % 16 == 0, "%s: stride %lld of %s is not a multiple of 16 bytes", name, s[i], what);
  return GPN_OK;
}

Strides strides(const long long* s) { return Strides{s[0], s[1], s[2]}; }

AttnP fill(const gpn_attn_args_t* x) {
  AttnP a = {};
  a.q = x->q, a.k = x->k, a.v = x->v, a.dout = x->dout;
  a.out = x->out, a.dq = x->dq, a.dk = x->dk, a.dv = x->dv;
  a.sq = strides(x->q_stride), a.sk = strides(x->k_stride), a.sv = strides(x->v_stride), a.sdo = strides(x->dout_stride);
  a.lse = x->lse, a.lengths = x->lengths, a.q_start = x->causal ? x->q_start : nullptr, a.key_mask = x->key_mask;
  a.mask_sb = x->key_mask_stride;
  a.B = x->B, a.Lq = x->Lq, a.Lk = x->Lk, a.Hq = x->Hq, a.Hkv = x->Hkv, a.D = x->D;
  a.G = x->Hq / x->Hkv, a.M = x->Lq * a.G;
  a.g_magic = a.G > 1 ? (unsigned)((0x100000000ull + a.G - 1) / a.G) : 0;
  a.causal = x->causal != 0, a.scale = x->scale, a.c = x->scale * LOG2E;
  return a;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

template <typename T, int DP>
int forward_t(AttnP& a, const Plan& pl, hipStream_t st) {
  constexpr bool F32 = sizeof(T) == 4;
  const long long grid = grid_of((long long)a.B * a.Hkv, (long long)pl.tiles * pl.nsplit);
  int rc;
  if (pl.few) {
    constexpr int KT = F32 && DP > 64 ? 16 : 32;  // four waves' keys and values of a stage: at most 76 KB
    using F = Fwd<T, DP, 1, 4, KT, 1>;
    rc = launch(k_attn_fwd<T, DP, 1, 4, KT, 1>, "k_attn_fwd", grid, F::NTH, F::lds, st, a);
  } else {
    constexpr int NB = F32 && DP > 64 ? 1 : 2;
    using F = Fwd<T, DP, 4, 1, 64, NB>;
    rc = launch(k_attn_fwd<T, DP, 4, 1, 64, NB>, "k_attn_fwd", grid, F::NTH, F::lds, st, a);
  }
  if (rc || pl.nsplit == 1) return rc;
  const long long rows = (long long)a.B * a.Hkv * a.M;
  return launch(k_attn_join<T>, "k_attn_join", (rows + 7) / 8, 256, 0, st, a);
}

// Keys of a workgroup of the dk / dv kernel: 4 waves' tiles.
int dkv_keys(bool f32) { return f32 ? 64 : 128; }

// Parts that the rows of a key tile are cut into: enough for two workgroups on every CU, with 256 rows or more each, so that a
// part's products outweigh its sums' way through memory.
int plan_dkv(const gpn_attn_args_t* x) {
  const long long M = (long long)x->Lq * (x->Hq / x->Hkv);
  const int bn = dkv_keys(x->dtype == GPN_DT_F32);
  long long tiles = (x->Lk + bn - 1) / bn;
  if (x->causal) tiles = (tiles + 1) / 2;
  const long long units = (long long)x->B * x->Hkv * tiles;
  if (units == 0 || units >= 256) return 1;
  long long s = 512 / units;
  if (s > M / 256) s = M / 256;
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

template <typename T, int DP>
int backward_t(AttnP& a, int nsplit, hipStream_t st) {
  constexpr bool F32 = sizeof(T) == 4;
  const long long prob = (long long)a.B * a.Hkv;
  {
    constexpr int KT = F32 && DP > 64 ? 32 : 64;
    using F = Dq<T, DP, 4, KT>;
    a.tiles = (a.M + F::BM - 1) / F::BM;
    const int rc = launch(k_attn_dq<T, DP, 4, KT>, "k_attn_dq", grid_of(prob, a.tiles), F::NTH, F::lds, st, a);
    if (rc) return rc;
  }
  using F = Dkv<T, DP, 4, 2>;
  static_assert(F::BN == (F32 ? 64 : 128) && F::lds <= 160 * 1024, "dkv_keys, LDS");
  a.tiles = (a.Lk + F::BN - 1) / F::BN, a.nsplit = nsplit;
  const long long units = (long long)(a.causal ? (a.tiles + 1) / 2 : a.tiles) * nsplit;
  const int rc = launch(k_attn_dkv<T, DP, 4, 2>, "k_attn_dkv", grid_of(prob, units), F::NTH, F::lds, st, a);
  if (rc || nsplit == 1) return rc;
  return launch(k_attn_dkv_join<T>, "k_attn_dkv_join", ((long long)a.B * a.Lk * a.Hkv * a.D / 2 + 255) / 256, 256, 0, st, a);
}

template <typename Fn>
int by_width(int D, Fn fn) {  // head widths are padded to the next of these with zeros
  if (D <= 16) return fn(std::integral_constant<int, 16>());
  if (D <= 32) return fn(std::integral_constant<int, 32>());
  if (D <= 64) return fn(std::integral_constant<int, 64>());
  if (D <= 96) return fn(std::integral_constant<int, 96>());
  return fn(std::integral_constant<int, 128>());
}

}  // namespace

extern "C" size_t gpn_attn_workspace_bytes(const gpn_attn_args_t* x, int backward) {
  if (check_args(x, "gpn_attn_workspace_bytes") || x->B == 0 || x->Lq == 0) return 0;
  const size_t rows = (size_t)x->B * x->Hq * x->Lq;
  if (backward) {  // delta, and the parts of dk and dv
    const int s = plan_dkv(x);
    return align256(rows * 4) + (s > 1 ? (size_t)s * 2 * x->B * x->Lk * x->Hkv * x->D * 4 : 0);
  }
  const Plan p = plan_forward(x);
  return p.nsplit == 1 ? 0 : align256(rows * p.nsplit * 4) + rows * p.nsplit * x->D * 4;
}

extern "C" int gpn_attn_forward(const gpn_attn_args_t* x, gpn_stream_t stream) {
  const char* name = "gpn_attn_forward";
  if (int rc = check_args(x, name)) return rc;
  if (x->B == 0 || x->Lq == 0) return GPN_OK;
  const int size = x->dtype == GPN_DT_F32 ? 4 : 2;
  if (int rc = check_tensor(x->q, x->q_stride, size, "q", name)) return rc;
  if (x->Lk > 0) {
    if (int rc = check_tensor(x->k, x->k_stride, size, "k", name)) return rc;
    if (int rc = check_tensor(x->v, x->v_stride, size, "v", name)) return rc;
  }
  if (int rc = check_tensor(x->out, nullptr, size, "out", name)) return rc;
  GPN_REQUIRE(x->lse, "%s: null lse", name);
  const Plan pl = plan_forward(x);
  const size_t need = gpn_attn_workspace_bytes(x, 0);
  GPN_REQUIRE(x->workspace_bytes >= need && (need == 0 || x->workspace), "%s: workspace of %zu bytes, %zu needed", name,
              x->workspace_bytes, need);
  AttnP a = fill(x);
  a.tiles = pl.tiles, a.nsplit = pl.nsplit, a.split_keys = pl.split_keys;
  if (pl.nsplit > 1) {
    a.part_l = (float*)x->workspace;
    a.part_o = (float*)((char*)x->workspace + align256((size_t)x->B * x->Hq * x->Lq * pl.nsplit * 4));
  }
  hipStream_t st = (hipStream_t)stream;
  return by_width(x->D, [&](auto dp) {
    return x->dtype == GPN_DT_F32 ? forward_t<float, decltype(dp)::value>(a, pl, st)
                                  : forward_t<bf16, decltype(dp)::value>(a, pl, st);
  });
}

extern "C" int gpn_attn_backward(const gpn_attn_args_t* x, gpn_stream_t stream) {
  const char* name = "gpn_attn_backward";
  if (int rc = check_args(x, name)) return rc;
  if (x->B == 0 || (x->Lq == 0 && x->Lk == 0)) return GPN_OK;
  const int size = x->dtype == GPN_DT_F32 ? 4 : 2;
  if (x->Lq > 0) {
    if (int rc = check_tensor(x->q, x->q_stride, size, "q", name)) return rc;
    if (int rc = check_tensor(x->dout, x->dout_stride, size, "dout", name)) return rc;
    if (int rc = check_tensor(x->out, nullptr, size, "out", name)) return rc;
    if (int rc = check_tensor(x->dq, nullptr, size, "dq", name)) return rc;
    GPN_REQUIRE(x->lse, "%s: null lse", name);
  }
  if (x->Lk > 0) {
    if (int rc = check_tensor(x->k, x->k_stride, size, "k", name)) return rc;
    if (int rc = check_tensor(x->v, x->v_stride, size, "v", name)) return rc;
    if (int rc = check_tensor(x->dk, nullptr, size, "dk", name)) return rc;
    if (int rc = check_tensor(x->dv, nullptr, size, "dv", name)) return rc;
  }
  const size_t need = gpn_attn_workspace_bytes(x, 1);
  GPN_REQUIRE(x->workspace_bytes >= need && (need == 0 || x->workspace), "%s: workspace of %zu bytes, %zu needed", name,
              x->workspace_bytes, need);
  AttnP a = fill(x);
  const int nsplit = plan_dkv(x);
  a.delta = (float*)x->workspace;
  a.part_o = (float*)((char*)x->workspace + align256((size_t)x->B * x->Hq * x->Lq * 4));
  hipStream_t st = (hipStream_t)stream;
  return by_width(x->D, [&](auto dp) {
    return x->dtype == GPN_DT_F32 ? backward_t<float, decltype(dp)::value>(a, nsplit, st)
                                  : backward_t<bf16, decltype(dp)::value>(a, nsplit, st);
  });
}
