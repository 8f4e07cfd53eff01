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
#include <algorithm>
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

constexpr int MAX_SPLIT = 64;
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
  // product with 8 bits, which is what its other operand has; their sums stay fp32.  Independent errors of half a step per
  // operand come to about what the gradients' own store to bf16 adds: 0.0024 of a gradient's norm, 0.0017 with operands in fp32
  // (4096 x 128 rays; 0.0029 where few keys are seen).
  static __device__ __forceinline__ Frag pack(const Acc& s, int t) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (bf16)s[8 * t + i];
    return f;
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
};

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

// ------------------------------------------------------------------------------------------------------ tiles in LDS
// A tile is rows of CPS 16-byte chunks without padding (the loads below write 1 KB runs), in an order that both ways of
// reading it find without bank conflicts: row r lies at phys(r), its chunk c in slot c ^ swz(phys(r)).  Sixteen rows read at one
// chunk (rowfrag) and four rows read at four neighbouring chunks (colfrag) both touch 64 different banks.  phys is the
// identity for bf16, whose column reads take four neighbouring rows; fp32 takes the rows 4h + i of the four lane groups h at
// once, so there the two low bit pairs of the row are exchanged.
constexpr int pow2_up(int x) { return x <= 2 ? 2 : x <= 4 ? 4 : x <= 8 ? 8 : x <= 16 ? 16 : 32; }

template <typename T, int DP>
struct Lay {
  using M = Mt<T>;
  static constexpr int CPS = pow2_up(DP / M::EP), ROWB = CPS * 16, HG = 64 / M::TM;
  static constexpr int DV = sizeof(T) == 2 && DP < 32 ? 32 : DP, MD = DV / M::TM, KF = DP / 16;
  static __device__ __forceinline__ int phys(int r) { return sizeof(T) == 2 ? r : (r & ~15) | (r & 3) << 2 | (r >> 2 & 3); }
  static __device__ __forceinline__ int swz(int p) {
    return ROWB == 32 ? p >> 3 & 1 : ROWB == 64 ? p >> 2 & 3 : ROWB == 128 ? (p >> 1 & 1) << 2 | (p >> 2 & 3) : (p & 3) << 2 | (p >> 2 & 3);
  }
  // 16 steps of k along d: fragment f of the row that the lane's column index names (rows n .. of a tile at x)
  static __device__ __forceinline__ typename M::Frag rowfrag(const char* x, int f, int lane) {
    const int p = phys(lane & (M::TM - 1)), c = HG * f + lane / M::TM;
    return *(const typename M::Frag*)(x + p * ROWB + (c ^ swz(p)) * 16);
  }
  // column tile md of the 16 rows at x, in the order of an accumulator's rows
  static __device__ __forceinline__ typename M::Frag colfrag(const char* x, int md, int lane) {
    if constexpr (sizeof(T) == 2) {
      // ds_read_b64_tr_b16: lanes 4j .. 4j+3 of a group of 16 address 16 columns of row j; lane l receives column l of the
      // four.  (Of a 16-wide head only half the tile's columns exist; the other lanes read the first half again, unused.)
      const int r = 4 * (lane >> 5) + (lane >> 2 & 3), c = (4 * md + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) & (CPS - 1);
      typedef __attribute__((address_space(3))) s4v* lp;
      const char* q = x + 8 * (lane & 1);
      const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + r * ROWB + (c ^ swz(r)) * 16));
      const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + (r + 8) * ROWB + (c ^ swz(r + 8)) * 16));
      return __builtin_bit_cast(typename M::Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int h = lane >> 4, c = 4 * md + (lane >> 2 & 3);
      typename M::Frag f;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = *(const float*)(x + (4 * i + h) * ROWB + (c ^ swz(4 * i + h)) * 16 + 4 * (lane & 3));
      return f;
    }
  }
};

__device__ __attribute__((aligned(16))) unsigned attn_zero[4];  // what hidden rows are read from
__device__ float attn_inf = INFINITY;

// Asynchronous loads into LDS: lane i's 16 (4) bytes land at lds + 16 i (4 i).  They count as vector memory loads, complete in
// order, and are waited for by the s_waitcnt of stage_done().
__device__ __forceinline__ void dma16(const void* p, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(p), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma16(const void* base, unsigned off, unsigned lds) {  // wave-uniform base
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(off), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma4(const void* p, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(p), "s"(lds) : "memory");
}
// The wave's own loads but the newest N have landed and its LDS reads are done; BAR: so have the other waves' of the workgroup.
template <int N, bool BAR>
__device__ __forceinline__ void stage_done() {
  if (BAR) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(size_t)(__attribute__((address_space(3))) const char*)p;
}

// ROWS rows of a tile, loaded by NW waves: which of its rows and chunks this lane brings.  A round is one load of every wave
// (STEP rows); row order and swizzle repeat every 16 rows, so NV rounds cover all different offsets.
template <typename T, int DP, int ROWS, int NW>
struct Dma {
  using L = Lay<T, DP>;
  static constexpr int RPI = 64 / L::CPS, STEP = RPI * NW, NI = ROWS <= STEP ? 1 : ROWS / STEP, NV = STEP >= 16 ? 1 : 16 / STEP;
  static_assert(ROWS % RPI == 0 && (ROWS <= STEP || ROWS % STEP == 0) && (NI == 1 || NI % NV == 0), "whole rounds");
  static constexpr int COUNT = NI;  // loads per wave and tile (none for a wave beyond ROWS)
  static __device__ __forceinline__ int place(int w, int lane, int i) { return (i * NW + w) * RPI + lane / L::CPS; }
  static __device__ __forceinline__ int row(int w, int lane, int i) { return L::phys(place(w, lane, i)); }  // phys is its own inverse
  static __device__ __forceinline__ int chunk(int w, int lane, int i) { return (lane & (L::CPS - 1)) ^ L::swz(place(w, lane, i)); }
  // all rows are there: uniform base + the lane's offset
  static __device__ __forceinline__ void whole(const T* base, long long stride, int D, unsigned lds, int w, int lane) {
    if (ROWS < STEP && w * RPI >= ROWS) return;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int v = i % NV, c = chunk(w, lane, v);
      const unsigned off = (unsigned)(row(w, lane, v) * (int)stride * (int)sizeof(T) + c * 16);
      if (c * Mt<T>::EP < D) dma16(base + (long long)(i / NV * NV * STEP) * stride, off, lds + (i * NW + w) * 1024);
    }
  }
  // uniform base + off(r) elements where there(r), else zero; 32-bit offsets
  template <typename Off, typename There>
  static __device__ __forceinline__ void near(const T* base, Off off, There there, int D, unsigned lds, int w, int lane) {
    if (ROWS < STEP && w * RPI >= ROWS) return;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = chunk(w, lane, i), r = row(w, lane, i);
      const char* p = (const char*)base + (unsigned)((off(r) + c * Mt<T>::EP) * (int)sizeof(T));
      if (c * Mt<T>::EP < D) dma16(there(r) ? (const void*)p : (const void*)attn_zero, lds + (i * NW + w) * 1024);
    }
  }
  // rows by address: at(r) is the row, or null for one that reads as zero
  template <typename At>
  static __device__ __forceinline__ void rows(At at, int D, unsigned lds, int w, int lane) {
    if (ROWS < STEP && w * RPI >= ROWS) return;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = chunk(w, lane, i);
      const T* p = at(row(w, lane, i));
      if (c * Mt<T>::EP < D) dma16(p ? (const void*)(p + c * Mt<T>::EP) : (const void*)attn_zero, lds + (i * NW + w) * 1024);
    }
  }
};

// A head narrower than DP: its last chunks are never loaded, and a product's zero times whatever stands there has to be zero.
// `rows` rows of tiles that follow each other from lds on.
template <typename T, int DP>
__device__ __forceinline__ void clear_tail(char* lds, int rows, int D, int nth) {
  using L = Lay<T, DP>;
  const int c0 = D / Mt<T>::EP, nc = DP / Mt<T>::EP - c0;
  if (nc <= 0) return;
  for (int i = threadIdx.x; i < rows * nc; i += nth) {
    const int r = i / nc, c = c0 + i - r * nc;
    *(u4v*)(lds + r * L::ROWB + (c ^ L::swz(r)) * 16) = u4v{0, 0, 0, 0};
  }
  __syncthreads();
}

struct Strides {
  long long b, l, h;
};

struct AttnP {
  const void *q, *k, *v, *dout;
  void *out, *dq, *dk, *dv;
  Strides sq, sk, sv, sdo;
  float *lse, *lse2, *delta, *part_o, *part_l;
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

// A use of loaded values before a loop of asynchronous loads: the compiler, which knows nothing of those, would else wait for
// its own loads at their first use inside the loop, in every turn, and with them for the stage just requested.
template <typename F, int N>
__device__ __forceinline__ void settle(F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// load_frags at a wave-uniform base + the lane's 32-bit offset (elements)
template <typename T, int KF>
__device__ __forceinline__ void load_frags_near(typename Mt<T>::Frag (&f)[KF], const T* base, int off, bool there, int D, int h) {
#pragma unroll
  for (int i = 0; i < KF; ++i) {
    const int d = 16 * i + Mt<T>::EP * h;
    u4v x = {0, 0, 0, 0};
    if (there && d < D) x = *(const u4v*)((const char*)base + (unsigned)((off + d) * (int)sizeof(T)));
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

// Which keys of a stage (KT <= 64 from j0 on) are there: bit x = key j0 + x.  With a mask its bytes are read a stage ahead.
template <int KT>
struct Keys {
  static constexpr unsigned long long ALL = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
  const unsigned char* km;
  int kend;
  unsigned char byte;
  __device__ __forceinline__ void fetch(int j0, int lane) {
    if (km) byte = lane < KT && j0 + lane < kend ? km[j0 + lane] : 0;
  }
  __device__ __forceinline__ unsigned long long bits(int j0) const {
    if (km) return __ballot(byte != 0);
    const int n = kend - j0;
    return n >= KT ? ALL : n <= 0 ? 0ull : (1ull << n) - 1;
  }
};

// The tile's rows of keys or values -> LDS; hidden rows are zero and never read (they may hold anything).
template <typename T, int DP, int KT, int NW>
__device__ __forceinline__ void load_keys(const T* base, long long stride, int D, int j0, unsigned long long bits, unsigned lds, int w,
                                          int lane) {
  using Dm = Dma<T, DP, KT, NW>;
  const T* b = base + (long long)j0 * stride;
  if (bits == Keys<KT>::ALL && stride < (1 << 22)) Dm::whole(b, stride, D, lds, w, lane);
  else Dm::rows([&](int r) { return bits >> r & 1 ? b + (long long)r * stride : (const T*)nullptr; }, D, lds, w, lane);
}

// bits of a stage -> the lane's: bit x = its row sees key j0 + x; shifted so that an accumulator's rows are at constant places
template <int KT>
__device__ __forceinline__ unsigned long long lane_bits(unsigned long long bits, int j0, int lim, int h) {
  if (lim < j0 + KT - 1) bits &= lim < j0 ? 0ull : ~0ull >> (63 - (lim - j0));
  return bits >> (4 * h);
}

// One stage of the forward: KT keys at ks / vs against the wave's rows.
template <typename T, int DP, int KT>
__device__ __forceinline__ void attend(const char* ks, const char* vs, const typename Mt<T>::Frag (&qf)[DP / 16],
                                       typename Mt<T>::Acc (&o)[Lay<T, DP>::MD], float& m, float& l, unsigned long long bits, int j0,
                                       int lim, float c, int lane) {
  using M = Mt<T>;
  using L = Lay<T, DP>;
  constexpr int TM = M::TM, MT = KT / TM;
  typename M::Acc sc[MT];
  __builtin_amdgcn_s_setprio(1);  // the wave that feeds the matrix unit goes first (2 x 4096 causal: 151 -> 145 us)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    sc[mt] = (typename M::Acc)(0.f);
#pragma unroll
    for (int f = 0; f < L::KF; ++f) sc[mt] = M::mma(L::rowfrag(ks + mt * TM * L::ROWB, f, lane), qf[f], sc[mt]);
  }
  __builtin_amdgcn_s_setprio(0);
  if (bits != Keys<KT>::ALL || __any(lim < j0 + KT - 1)) {
    bits = lane_bits<KT>(bits, j0, lim, lane / TM);
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
  const bool grow = (mx - m) * c > 8.f;  // of a row without a key so far: inf > 8; still without: nan > 8
  if (__any(grow)) {
    const float alpha = grow ? exp2_((m - mx) * c) : 1.f;
    m = grow ? mx : m;
    l *= alpha;
#pragma unroll
    for (int md = 0; md < L::MD; ++md) o[md] *= alpha;
  }
  const float mc = m == -INFINITY ? 0.f : m * c;
  float sum = 0.f;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int r = 0; r < M::NC; ++r) {
      const float e = exp2_(__builtin_fmaf(sc[mt][r], c, -mc));
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
      for (int md = 0; md < L::MD; ++md)
        o[md] = M::mma(L::colfrag(vs + (mt * TM + 16 * t) * L::ROWB, md, lane), pf, o[md]);
    }
}

extern __shared__ __attribute__((aligned(1024))) char attn_smem[];

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// what a forward workgroup needs to know of its rows
struct Rows {
  int row, i, g, hq, lim, kbeg, kend;
  bool live;
};
__device__ __forceinline__ Rows rows_of(const AttnP& a, const Prob& p, int row0, int row, int nrows, int split) {
  Rows r;
  r.row = row, r.live = row < a.M;
  r.i = row_pos(a, r.live ? row : 0), r.g = (r.live ? row : 0) - r.i * a.G, r.hq = p.hk * a.G + r.g;
  r.lim = a.causal ? p.qs + r.i : INT_MAX;  // last key the row may see
  r.kbeg = 0, r.kend = p.len;
  if (a.causal) r.kend = min(r.kend, p.qs + row_pos(a, min(row0 + nrows, a.M) - 1) + 1);
  if (a.nsplit > 1) r.kbeg = split * a.split_keys, r.kend = min(r.kend, r.kbeg + a.split_keys);
  return r;
}

// ---------------------------------------------------------------------------------------------------- forward
// NW waves with TM rows each share stages of KT keys and values: while one stage is worked on, the next lands in LDS.  WK = 2:
// twice as many waves, each with half of every stage's keys, whose sums are joined in LDS (is_mid has the rule).
// Bound by the matrix and vector instructions of a wave, which overlap as far as two waves per SIMD do: 8192 causal positions, 32
// query heads on 8 of 128, bf16: 543 us, 1010 TFLOP/s of the visible pairs (a library product reaches 1180 to 1320); 4 x 4096, 16
// heads of 64: 345 us, 800 TFLOP/s (half the products per exponential); fp32 2 x 1024, 8 heads of 128: 95 us, 90 of 153 TFLOP/s, one
// wave per SIMD.  A third stage in LDS changes nothing: the loads are not what it waits for.
template <typename T, int DP, int NW, int KT>
struct Fwd {
  using L = Lay<T, DP>;
  static constexpr int TM = Mt<T>::TM, BM = NW * TM, NTH = 64 * NW, TILE = KT * L::ROWB;
  static constexpr size_t lds = 4 * TILE;  // two stages of keys and values
};

template <typename T, int DP, int NW, int WK, int KT>
__global__ void __launch_bounds__(64 * NW * WK, 2) k_attn_fwd(const AttnP a) {
  using F = Fwd<T, DP, NW, KT>;
  using M = Mt<T>;
  using L = Lay<T, DP>;
  constexpr int KW = KT / WK;  // the wave's share of a stage
  int pr, unit;
  if (!locate(a.B * a.Hkv, a.tiles * a.nsplit, pr, unit)) return;
  // causal: the longest tiles first; where all are on the card at once (two per CU), the second half in turn, shortest beside
  // longest
  const int split = unit / a.tiles, u = unit - split * a.tiles, most = WK == 2 ? (a.tiles + 1) / 2 : a.tiles;
  const int tile = u < most ? a.tiles - 1 - u : u - most;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = wave_index(), wm = wave % NW, wk = wave / NW, n = lane & (M::TM - 1), h = lane / M::TM;
  const Rows r = rows_of(a, p, tile * F::BM, tile * F::BM + wm * M::TM + n, F::BM, split);
  clear_tail<T, DP>(attn_smem, 4 * KT, a.D, F::NTH * WK);

  const T* kb = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* vb = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const unsigned base = lds_address(attn_smem);
  Keys<KT> keys = {a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr, r.kend, 0};
  const auto request = [&](int j0, unsigned long long bits, int buf) {
    load_keys<T, DP, KT, NW * WK>(kb, a.sk.l, a.D, j0, bits, base + buf * 2 * F::TILE, wave, lane);
    load_keys<T, DP, KT, NW * WK>(vb, a.sv.l, a.D, j0, bits, base + (buf * 2 + 1) * F::TILE, wave, lane);
  };
  keys.fetch(r.kbeg, lane);
  unsigned long long bits = keys.bits(r.kbeg), next = 0;
  if (bits) request(r.kbeg, bits, 0);
  keys.fetch(r.kbeg + KT, lane);

  typename M::Frag qf[L::KF];
  load_frags<T, L::KF>(qf, r.live ? (const T*)a.q + p.b * a.sq.b + r.i * a.sq.l + r.hq * a.sq.h : nullptr, a.D, h);
  typename M::Acc o[L::MD];
#pragma unroll
  for (int md = 0; md < L::MD; ++md) o[md] = (typename M::Acc)(0.f);
  float m = -INFINITY, l = 0.f;  // reference of the raw scores; this lane's share of the sum
  settle(qf);
  stage_done<0, true>();
  int buf = 0;
  for (int j0 = r.kbeg; j0 < r.kend; j0 += KT, buf ^= 1, bits = next) {
    next = keys.bits(j0 + KT);
    keys.fetch(j0 + 2 * KT, lane);
    if (next) request(j0 + KT, next, buf ^ 1);
    const char* ks = attn_smem + buf * 2 * F::TILE + wk * KW * L::ROWB;
    const unsigned long long mine = bits >> (wk * KW) & Keys<KW>::ALL;
    if (mine && !__all(r.lim < j0 + wk * KW)) attend<T, DP, KW>(ks, ks + F::TILE, qf, o, m, l, mine, j0 + wk * KW, r.lim, a.c, lane);
    stage_done<0, true>();
  }
  l = col_sum<T>(l);
  if constexpr (WK == 2) {  // the waves of the other half of every stage hand reference, sum and output over
    float* mo = (float*)attn_smem + NW * L::MD * M::NC * 64;
    fl4* x = (fl4*)attn_smem + wm * L::MD * (M::NC / 4) * 64 + lane;
    if (wk) {
      mo[wm * 64 + lane] = m, mo[(NW + wm) * 64 + lane] = l;
#pragma unroll
      for (int md = 0; md < L::MD; ++md)
#pragma unroll
        for (int q = 0; q < M::NC / 4; ++q) {
          fl4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = o[md][4 * q + e];
          x[(md * (M::NC / 4) + q) * 64] = y;
        }
    }
    __syncthreads();
    if (wk) return;
    const float m1 = mo[wm * 64 + lane], l1 = mo[(NW + wm) * 64 + lane], mm = fmaxf(m, m1), ms = mm == -INFINITY ? 0.f : mm;
    const float f0 = exp2_((m - ms) * a.c), f1 = exp2_((m1 - ms) * a.c);
    m = mm, l = l * f0 + l1 * f1;
#pragma unroll
    for (int md = 0; md < L::MD; ++md)
#pragma unroll
      for (int q = 0; q < M::NC / 4; ++q) {
        const fl4 y = x[(md * (M::NC / 4) + q) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[md][4 * q + e] = o[md][4 * q + e] * f0 + y[e] * f1;
      }
  }
  if (!r.live) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row without a key is zero
  const float l2 = l == 0.f ? -INFINITY : m * a.c + log2_(l);
  if (a.nsplit > 1) {
    const long long at = ((long long)split * a.B * a.Hkv + pr) * a.M + r.row;
    if (h == 0) a.part_l[at] = l2;
    store_cols<T, float, L::MD>(o, inv, a.part_o + at * a.D, a.D, h);
    return;
  }
  if (h == 0) a.lse[((long long)p.b * a.Hq + r.hq) * a.Lq + r.i] = l2 * LN2;
  store_cols<T, T, L::MD>(o, inv, (T*)a.out + (((long long)p.b * a.Lq + r.i) * a.Hq + r.hq) * a.D, a.D, h);
}

// Up to KB keys (the samples of a ray): all of them are loaded at once and a row's softmax is taken in one piece.
// Bound by memory: 4096 rays of 64 samples, 4 fp32 heads of 16: 66 us, 4.1 TB/s of its own bytes (a large copy: 4.8); 4096 x 128 in
// bf16, with four times the scores, 95 us, 2.8 TB/s, bound by their vector instructions.  Workgroups that stay and load the next ray ahead took longer (90 against 74 us): the waves of other rays
// on the CU hide a ray's loads better.
template <typename T, int DP, int NW, int KB>
struct OnePiece {
  using L = Lay<T, DP>;
  static constexpr int TM = Mt<T>::TM, BM = NW * TM, NTH = 64 * NW, TILE = KB * L::ROWB;
  static constexpr size_t lds = 2 * TILE;
};

template <typename T, int DP, int NW, int KB>
__global__ void __launch_bounds__(64 * NW, 2) k_attn_one_piece(const AttnP a) {
  using F = OnePiece<T, DP, NW, KB>;
  using M = Mt<T>;
  using L = Lay<T, DP>;
  using Dm = Dma<T, DP, KB, NW>;
  constexpr int TM = M::TM, MT = KB / TM, WORDS = KB / 64;
  int pr, tile;
  if (!locate(a.B * a.Hkv, a.tiles, pr, tile)) return;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = wave_index(), n = lane & (TM - 1), h = lane / TM;
  const Rows r = rows_of(a, p, tile * F::BM, tile * F::BM + wave * TM + n, F::BM, 0);
  clear_tail<T, DP>(attn_smem, 2 * KB, a.D, F::NTH);

  const T* kb = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* vb = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const unsigned char* km = a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr;
  const unsigned base = lds_address(attn_smem);
  unsigned long long bits[WORDS];
  bool all = true;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int j = 64 * w + lane;
    bits[w] = __ballot(j < r.kend && (!km || km[j]));
    all &= bits[w] == ~0ull;
  }
  if (all && max(a.sk.l, a.sv.l) < (1 << 22)) {
    Dm::whole(kb, a.sk.l, a.D, base, wave, lane);
    Dm::whole(vb, a.sv.l, a.D, base + F::TILE, wave, lane);
  } else {
    const auto there = [&](int j) { return bits[WORDS == 1 ? 0 : j >> 6] >> (j & 63) & 1; };
    Dm::rows([&](int j) { return there(j) ? kb + j * a.sk.l : (const T*)nullptr; }, a.D, base, wave, lane);
    Dm::rows([&](int j) { return there(j) ? vb + j * a.sv.l : (const T*)nullptr; }, a.D, base + F::TILE, wave, lane);
  }
  typename M::Frag qf[L::KF];
  load_frags<T, L::KF>(qf, r.live ? (const T*)a.q + p.b * a.sq.b + r.i * a.sq.l + r.hq * a.sq.h : nullptr, a.D, h);
  stage_done<0, true>();

  typename M::Acc sc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    sc[mt] = (typename M::Acc)(0.f);
#pragma unroll
    for (int f = 0; f < L::KF; ++f) sc[mt] = M::mma(L::rowfrag(attn_smem + mt * TM * L::ROWB, f, lane), qf[f], sc[mt]);
  }
  if (!all || __any(r.lim < KB - 1)) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const unsigned long long lb = lane_bits<64>(bits[w], 64 * w, r.lim, h);
#pragma unroll
      for (int mt = w * 64 / TM; mt < (w + 1) * 64 / TM; ++mt)
#pragma unroll
        for (int x = 0; x < M::NC; ++x)
          if (!(lb >> (mt * TM - 64 * w + M::crow(x, 0)) & 1)) sc[mt][x] = -INFINITY;
    }
  }
  float m = sc[0][0];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int x = 0; x < M::NC; ++x) m = fmaxf(m, sc[mt][x]);
  m = col_max<T>(m);
  const float mc = m == -INFINITY ? 0.f : m * a.c;
  float l = 0.f;
  typename M::Acc o[L::MD];
#pragma unroll
  for (int md = 0; md < L::MD; ++md) o[md] = (typename M::Acc)(0.f);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int x = 0; x < M::NC; ++x) {
      sc[mt][x] = exp2_(__builtin_fmaf(sc[mt][x], a.c, -mc));
      l += sc[mt][x];
    }
#pragma unroll
    for (int t = 0; t < TM / 16; ++t) {
      const typename M::Frag pf = M::pack(sc[mt], t);
#pragma unroll
      for (int md = 0; md < L::MD; ++md)
        o[md] = M::mma(L::colfrag(attn_smem + F::TILE + (mt * TM + 16 * t) * L::ROWB, md, lane), pf, o[md]);
    }
  }
  l = col_sum<T>(l);
  if (!r.live) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row without a key is zero
  if (h == 0) a.lse[((long long)p.b * a.Hq + r.hq) * a.Lq + r.i] = (l == 0.f ? -INFINITY : m * a.c + log2_(l)) * LN2;
  store_cols<T, T, L::MD>(o, inv, (T*)a.out + (((long long)p.b * a.Lq + r.i) * a.Hq + r.hq) * a.D, a.D, h);
}

// Few rows (new tokens of sequences, or too few tiles to fill the card): the WK waves share a tile of rows and divide the keys,
// each with stages of its own and no barrier until their sums are joined.
// Bound by memory for long keys: one query for each of 8 sequences of 16 K keys, 32 heads on 8 of 128, bf16: 107 us, 5.0 TB/s; fp32:
// 202 us, 5.3 TB/s; with lengths from 0 to 16 K 74 us in bf16.  One query against 257 keys: 7 us, the latency of three loads in a row.
template <typename T, int DP, int WK, int KT>
struct Few {
  using L = Lay<T, DP>;
  static constexpr int TM = Mt<T>::TM, NTH = 64 * WK, TILE = KT * L::ROWB, LO = L::DV + 4;
  static constexpr size_t stage_bytes = (size_t)WK * 4 * TILE, join_bytes = (size_t)WK * TM * (LO + 2) * 4;
  static constexpr size_t lds = stage_bytes > join_bytes ? stage_bytes : join_bytes;
};

template <typename T, int DP, int WK, int KT>
__global__ void __launch_bounds__(64 * WK, 2) k_attn_few(const AttnP a) {
  using F = Few<T, DP, WK, KT>;
  using M = Mt<T>;
  using L = Lay<T, DP>;
  constexpr int TM = M::TM, LO = F::LO;
  int pr, unit;
  if (!locate(a.B * a.Hkv, a.tiles * a.nsplit, pr, unit)) return;
  const int split = unit / a.tiles, row0 = (a.tiles - 1 - (unit - split * a.tiles)) * TM;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = wave_index(), n = lane & (TM - 1), h = lane / TM;
  const Rows r = rows_of(a, p, row0, row0 + n, TM, split);
  clear_tail<T, DP>(attn_smem, WK * 4 * KT, a.D, F::NTH);

  const T* kb = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* vb = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const char* mine = attn_smem + wave * 4 * F::TILE;
  const unsigned base = lds_address(attn_smem) + wave * 4 * F::TILE;
  Keys<KT> keys = {a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr, r.kend, 0};
  const auto request = [&](int j0, unsigned long long bits, int buf) {
    load_keys<T, DP, KT, 1>(kb, a.sk.l, a.D, j0, bits, base + buf * 2 * F::TILE, 0, lane);
    load_keys<T, DP, KT, 1>(vb, a.sv.l, a.D, j0, bits, base + (buf * 2 + 1) * F::TILE, 0, lane);
  };
  // two stages on their way: the second lands while the first is worked on, whose memory the third then takes.  With a key mask one:
  // the compiler, which does not count these loads, waits for all of them where it waits for the mask's bytes.
  constexpr int NEXT = WK * KT, LOADS = 2 * Dma<T, DP, KT, 1>::COUNT;
  const int jb = r.kbeg + wave * KT;
  keys.fetch(jb, lane);
  unsigned long long bits = keys.bits(jb);
  keys.fetch(jb + NEXT, lane);
  if (bits) request(jb, bits, 0);
  unsigned long long next = keys.bits(jb + NEXT), after;
  keys.fetch(jb + 2 * NEXT, lane);
  if (next) request(jb + NEXT, next, 1);
  typename M::Frag qf[L::KF];
  load_frags<T, L::KF>(qf, r.live ? (const T*)a.q + p.b * a.sq.b + r.i * a.sq.l + r.hq * a.sq.h : nullptr, a.D, h);
  typename M::Acc o[L::MD];
#pragma unroll
  for (int md = 0; md < L::MD; ++md) o[md] = (typename M::Acc)(0.f);
  float m = -INFINITY, l = 0.f;
  settle(qf);
  int buf = 0;
  for (int j0 = jb; j0 < r.kend; j0 += NEXT, buf ^= 1, bits = next, next = after) {
    if (next) stage_done<LOADS, false>();
    else stage_done<0, false>();
    if (bits && !__all(r.lim < j0))
      attend<T, DP, KT>(mine + buf * 2 * F::TILE, mine + (buf * 2 + 1) * F::TILE, qf, o, m, l, bits, j0, r.lim, a.c, lane);
    after = keys.bits(j0 + 2 * NEXT);
    keys.fetch(j0 + 3 * NEXT, lane);
    if (after) {
      stage_done<63, false>();  // the stage has been read (no wait for the loads)
      request(j0 + 2 * NEXT, after, buf);
    }
  }
  stage_done<0, false>();
  l = col_sum<T>(l);

  float* mo = (float*)attn_smem;  // [WK][TM] references, [WK][TM] sums, [WK][TM][LO] outputs
  float* lo = mo + WK * TM;
  float* oo = lo + WK * TM;
  __syncthreads();  // every wave is past its last stage
  if (h == 0) mo[wave * TM + n] = m, lo[wave * TM + n] = l;
#pragma unroll
  for (int md = 0; md < L::MD; ++md)
#pragma unroll
    for (int q = 0; q < M::NC / 4; ++q) {
      fl4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = o[md][4 * q + e];
      *(fl4*)(oo + (wave * TM + n) * LO + md * TM + M::crow(4 * q, h)) = x;
    }
  __syncthreads();
  for (int x = threadIdx.x; x < TM * (DP / 4); x += F::NTH) {
    const int rt = x / (DP / 4), rw = row0 + rt, d = 4 * (x % (DP / 4));
    if (rw >= a.M) continue;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; ++w) mm = fmaxf(mm, mo[w * TM + rt]);
    const float ms = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    fl4 acc = (fl4)(0.f);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float f = exp2_((mo[w * TM + rt] - ms) * a.c);
      ll += f * lo[w * TM + rt];
      acc += f * *(const fl4*)(oo + (w * TM + rt) * LO + d);
    }
    acc *= ll > 0.f || ll != ll ? 1.f / ll : 0.f;
    const float l2 = ll == 0.f ? -INFINITY : ms * a.c + log2_(ll);
    const int i = row_pos(a, rw), hq = p.hk * a.G + rw - i * a.G;
    if (a.nsplit > 1) {
      const long long at = ((long long)split * a.B * a.Hkv + pr) * a.M + rw;
      if (d == 0) a.part_l[at] = l2;
      if (d < a.D) *(fl4*)(a.part_o + at * a.D + d) = acc;
    } else {
      if (d == 0) a.lse[((long long)p.b * a.Hq + hq) * a.Lq + i] = l2 * LN2;
      typedef T V4 __attribute__((ext_vector_type(4)));
      V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)acc[e];
      if (d < a.D) *(V4*)((T*)a.out + (((long long)p.b * a.Lq + i) * a.Hq + hq) * a.D + d) = y;
    }
  }
}

// Joins the splits of a row: every split left its own normalised output and log2-sum-exp.  32 lanes per row, 4 values a lane;
// lane s first looks at the splits s and s + 32.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_join(const AttnP a) {
  static_assert(MAX_SPLIT <= 64, "two splits per lane");
  const long long rows = (long long)a.B * a.Hkv * a.M, x = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int s0 = threadIdx.x & 31, d = 4 * s0;
  const long long xr = x < rows ? x : rows - 1;
  const float la = s0 < a.nsplit ? a.part_l[s0 * rows + xr] : -INFINITY;
  const float lb = s0 + 32 < a.nsplit ? a.part_l[(s0 + 32) * rows + xr] : -INFINITY;
  float mm = fmaxf(la, lb);
  bool bad = la != la || lb != lb;
#pragma unroll
  for (int k = 16; k; k >>= 1) mm = fmaxf(mm, __shfl_xor(mm, k)), bad |= __shfl_xor((int)bad, k) != 0;
  const float ms = mm == -INFINITY ? 0.f : mm;
  const float wa = exp2_(la - ms), wb = exp2_(lb - ms);
  float w = wa + wb;
#pragma unroll
  for (int k = 16; k; k >>= 1) w += __shfl_xor(w, k);
  fl4 acc = (fl4)(0.f);
  const float* o = a.part_o + xr * a.D + (d < a.D ? d : 0);
  for (int s = 0; s < a.nsplit; s += 8) {  // eight parts on their way at once; those behind the last have no weight
    fl4 y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = *(const fl4*)(o + min(s + k, a.nsplit - 1) * rows * a.D);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc += (s + k < a.nsplit ? __shfl(s < 32 ? wa : wb, (s + k) & 31, 32) : 0.f) * y[k];
  }
  if (x >= rows) return;
  const int pr = (int)(x / a.M), row = (int)(x - (long long)pr * a.M);
  const int b = pr / a.Hkv, i = row_pos(a, row), hq = (pr - b * a.Hkv) * a.G + row - i * a.G;
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
//   p = exp(s - lse), ds = p (do.v - delta), dq = scale sum ds k,  delta = do.o
// delta and the log-sum-exp in powers of two (+inf for a row without a key) are left for the other kernel.
// Bound like the forward: 4 x 4096, 16 heads of 64, bf16: 410 us, 1000 TFLOP/s; 2 x 4096 causal, 16 heads on 4 of 128: 203 us, 1020.
template <typename T, int DP, int NW, int KT, int WK>
__global__ void __launch_bounds__(64 * NW * WK, 2) k_attn_dq(const AttnP a) {
  using F = Fwd<T, DP, NW, KT>;
  using M = Mt<T>;
  using L = Lay<T, DP>;
  constexpr int TM = M::TM, MT = KT / TM / WK, NTH = 64 * NW * WK;
  static_assert(WK == 1 || WK == 2, "the join below is of two waves");
  int pr, unit;
  if (!locate(a.B * a.Hkv, a.tiles, pr, unit)) return;
  // longest tiles first; where all are on the card at once (two per CU), the second half in turn, shortest beside longest
  const int most = NW == 2 ? (a.tiles + 1) / 2 : a.tiles, tile = unit < most ? a.tiles - 1 - unit : unit - most;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = wave_index(), wm = wave % NW, wk = wave / NW, n = lane & (TM - 1), h = lane / TM;
  const Rows r = rows_of(a, p, tile * F::BM, tile * F::BM + wm * TM + n, F::BM, 0);
  clear_tail<T, DP>(attn_smem, 4 * KT, a.D, NTH);

  const T* kb = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* vb = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const unsigned base = lds_address(attn_smem);
  Keys<KT> keys = {a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr, r.kend, 0};
  const auto request = [&](int j0, unsigned long long bits, int buf) {
    load_keys<T, DP, KT, NW * WK>(kb, a.sk.l, a.D, j0, bits, base + buf * 2 * F::TILE, wave, lane);
    load_keys<T, DP, KT, NW * WK>(vb, a.sv.l, a.D, j0, bits, base + (buf * 2 + 1) * F::TILE, wave, lane);
  };
  keys.fetch(0, lane);
  unsigned long long bits = keys.bits(0), next = 0;
  if (bits) request(0, bits, 0);
  keys.fetch(KT, lane);

  typename M::Frag qf[L::KF], df[L::KF];
  load_frags<T, L::KF>(qf, r.live ? (const T*)a.q + p.b * a.sq.b + r.i * a.sq.l + r.hq * a.sq.h : nullptr, a.D, h);
  load_frags<T, L::KF>(df, r.live ? (const T*)a.dout + p.b * a.sdo.b + r.i * a.sdo.l + r.hq * a.sdo.h : nullptr, a.D, h);
  const long long at = ((long long)p.b * a.Hq + r.hq) * a.Lq + r.i, orow = (((long long)p.b * a.Lq + r.i) * a.Hq + r.hq) * a.D;
  float delta = 0.f;
  {
    typename M::Frag of[L::KF];
    load_frags<T, L::KF>(of, r.live ? (const T*)a.out + orow : nullptr, a.D, h);
#pragma unroll
    for (int f = 0; f < L::KF; ++f)
#pragma unroll
      for (int e = 0; e < M::EP; ++e) delta = __builtin_fmaf((float)df[f][e], (float)of[f][e], delta);
    delta = col_sum<T>(delta);
  }
  float lse2 = r.live ? a.lse[at] * LOG2E : INFINITY;
  if (lse2 == -INFINITY) lse2 = INFINITY;  // a row without a key: every probability is zero
  if (r.live && h == 0 && wk == 0) a.delta[(long long)pr * a.M + r.row] = delta, a.lse2[(long long)pr * a.M + r.row] = lse2;

  typename M::Acc dq[L::MD];
#pragma unroll
  for (int md = 0; md < L::MD; ++md) dq[md] = (typename M::Acc)(0.f);
  settle(qf), settle(df);
  asm volatile("" : "+v"(lse2), "+v"(delta));
  stage_done<0, true>();
  int buf = 0;
  for (int j0 = 0; j0 < r.kend; j0 += KT, buf ^= 1, bits = next) {
    next = keys.bits(j0 + KT);
    keys.fetch(j0 + 2 * KT, lane);
    if (next) request(j0 + KT, next, buf ^ 1);
    if (bits && !__all(r.lim < j0)) {
      const bool partly = bits != Keys<KT>::ALL || __any(r.lim < j0 + KT - 1);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const char* kt = attn_smem + buf * 2 * F::TILE + (wk * MT + mt) * TM * L::ROWB;
        const char* vt = kt + F::TILE;
        typename M::Acc sc = (typename M::Acc)(0.f), dp = (typename M::Acc)(0.f);
        if (sizeof(T) == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int f = 0; f < L::KF; ++f) {
          sc = M::mma(L::rowfrag(kt, f, lane), qf[f], sc);
          dp = M::mma(L::rowfrag(vt, f, lane), df[f], dp);
        }
        __builtin_amdgcn_s_setprio(0);
        if (partly) {  // a hidden score of -inf leaves a probability of zero
          const unsigned long long lb = lane_bits<KT>(bits, j0, r.lim, h) >> (wk * MT * TM);
#pragma unroll
          for (int x = 0; x < M::NC; ++x)
            if (!(lb >> (mt * TM + M::crow(x, 0)) & 1)) sc[x] = -INFINITY;
        }
#pragma unroll
        for (int x = 0; x < M::NC; ++x) sc[x] = exp2_(__builtin_fmaf(sc[x], a.c, -lse2)) * (dp[x] - delta);
#pragma unroll
        for (int t = 0; t < TM / 16; ++t) {
          const typename M::Frag sf = M::pack(sc, t);
#pragma unroll
          for (int md = 0; md < L::MD; ++md) dq[md] = M::mma(L::colfrag(kt + 16 * t * L::ROWB, md, lane), sf, dq[md]);
        }
      }
    }
    stage_done<0, true>();
  }
  if constexpr (WK == 2) {  // the waves of the other half of every stage hand their sums over
    fl4* x = (fl4*)attn_smem + wm * L::MD * (M::NC / 4) * 64 + lane;
#pragma unroll
    for (int md = 0; md < L::MD; ++md)
#pragma unroll
      for (int q = 0; q < M::NC / 4; ++q)
        if (wk) {
          fl4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = dq[md][4 * q + e];
          x[(md * (M::NC / 4) + q) * 64] = y;
        }
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int md = 0; md < L::MD; ++md)
#pragma unroll
      for (int q = 0; q < M::NC / 4; ++q) {
        const fl4 y = x[(md * (M::NC / 4) + q) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) dq[md][4 * q + e] += y[e];
      }
  }
  if (r.live) store_cols<T, T, L::MD>(dq, a.scale, (T*)a.dq + orow, a.D, h);
}

// ---------------------------------------------------------------------------------------------- gradients of keys, values
// Keys and values are stationary, a wave holds TM of them; the rows of all query heads that share them walk past, so the sum
// over the group is part of the walk and its order is fixed.  WN waves along the keys x WR waves along the rows: the WR waves of
// the same keys take the rows of a stage in turns and join their sums at the end, so that two waves fit a SIMD (256 registers)
// without a second copy of the keys' sums in memory.  Where those registers are short (VL) the values come from LDS; pairs of
// 128-wide bf16 heads still lack three, which lie in scratch.
// Work is cut evenly: under `causal` a workgroup takes the key tiles t and tiles - 1 - t, which together see as many rows as any
// other such pair, and every tile's own rows are cut into nsplit parts (fp32 sums in the workspace, joined in order).
// Bound by LDS as well: every row is read from there twice in each direction, for four products.  4 x 4096, 16 heads of 64, bf16:
// 620 us, 890 TFLOP/s; 2 x 4096 causal, 16 heads on 4 of 128: 309 us, 890.
template <typename T, int DP, int WN, int WR>
struct Dkv {
  using M = Mt<T>;
  using L = Lay<T, DP>;
  static constexpr int TM = M::TM, RW = sizeof(T) == 4 && DP > 64 ? 16 : 32, RB = WR * RW, MT = RW / TM, BN = WN * TM;
  static constexpr int NW = WN * WR, NTH = 64 * NW, TILE = RB * L::ROWB, STAGE = 2 * TILE, NBUF = WR == 1 && DP > 64 ? 2 : 3;
  static constexpr bool VL = DP > 64;
  static constexpr int stats_at = NBUF * STAGE, v_at = stats_at + NBUF * 512;  // [NBUF][2][64] floats; values
  static constexpr size_t stage_bytes = v_at + (VL ? BN * L::ROWB : 0);
  static constexpr size_t join_bytes = WR > 1 ? (size_t)WN * 2 * L::MD * M::NC * 64 * 4 : 0;
  static constexpr size_t lds = stage_bytes > join_bytes ? stage_bytes : join_bytes;
  static constexpr int LOADS = 2 * Dma<T, DP, RB, NW>::COUNT;  // of a wave per stage: this many or more, or (no rows for it) none
};

template <typename T, int DP, int WN, int WR>
__global__ void __launch_bounds__(64 * WN * WR, 2) k_attn_dkv(const AttnP a) {
  using F = Dkv<T, DP, WN, WR>;
  using M = Mt<T>;
  using L = Lay<T, DP>;
  static_assert(WR == 1 || WR == 2, "the join below exchanges between two waves");
  static_assert(F::RB <= 64, "one wave brings a stage's row statistics");
  constexpr int TM = F::TM, MT = F::MT, RB = F::RB, BN = F::BN, KF = L::KF, MD = L::MD, NW = F::NW;
  constexpr bool VL = F::VL;
  using Dm = Dma<T, DP, RB, NW>;
  int pr, unit;
  if (!locate(a.B * a.Hkv, (a.causal ? (a.tiles + 1) / 2 : a.tiles) * a.nsplit, pr, unit)) return;
  const int tu = unit / a.nsplit, split = unit - tu * a.nsplit;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = wave_index(), wn = wave % WN, wr = wave / WN;
  const int n = lane & (TM - 1), h = lane / TM;
  const unsigned char* km = a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr;
  const auto first_row = [&](int j) { return !a.causal || j <= p.qs ? 0 : j - p.qs >= a.Lq ? INT_MAX : (j - p.qs) * a.G; };
  const unsigned base = lds_address(attn_smem);
  const float* stats = (const float*)(attn_smem + F::stats_at);
  const char* vw = attn_smem + F::v_at + wn * TM * L::ROWB;

  // Where the group divides a round of loads (STEP rows), every lane's part of a row's address stays, and a stage is a uniform
  // base on top; else row by row.  Rows at and behind M are those of row M - 1 again, with a probability of zero.
  const bool even = Dm::NV == 1 && Dm::STEP % a.G == 0 && RB % a.G == 0 &&
                    max(a.sq.l, a.sdo.l) < (1 << 20) && max(a.sq.h, a.sdo.h) < (1 << 20);
  const int er = Dm::row(wave, lane, 0), ei = row_pos(a, er), eg = er - ei * a.G, ec = Dm::chunk(wave, lane, 0);
  const unsigned eq = (unsigned)((ei * (int)a.sq.l + eg * (int)a.sq.h) * (int)sizeof(T) + ec * 16);
  const unsigned ed = (unsigned)((ei * (int)a.sdo.l + eg * (int)a.sdo.h) * (int)sizeof(T) + ec * 16);
  const bool mine = RB >= Dm::STEP || wave * Dm::RPI < RB, there = ec * M::EP < a.D;
  const T* q0 = (const T*)a.q + p.b * a.sq.b + (long long)p.hk * a.G * a.sq.h;
  const T* d0 = (const T*)a.dout + p.b * a.sdo.b + (long long)p.hk * a.G * a.sdo.h;
  const auto request = [&](int r0, int buf) {
    const unsigned to = base + buf * F::STAGE;
    if (even && r0 + RB <= a.M) {
      const int i0 = row_pos(a, r0), is = Dm::STEP / a.G;
      if (mine && there) {
#pragma unroll
        for (int i = 0; i < Dm::NI; ++i) {
          dma16(q0 + (long long)(i0 + i * is) * a.sq.l, eq, to + (i * NW + wave) * 1024);
          dma16(d0 + (long long)(i0 + i * is) * a.sdo.l, ed, to + F::TILE + (i * NW + wave) * 1024);
        }
      }
    } else {
      const auto at = [&](const T* x, const Strides& s, int r) {
        r = min(r0 + r, a.M - 1);
        const int i = row_pos(a, r);
        return x + i * s.l + (r - i * a.G) * s.h;
      };
      Dm::rows([&](int r) { return at(q0, a.sq, r); }, a.D, to, wave, lane);
      Dm::rows([&](int r) { return at(d0, a.sdo, r); }, a.D, to + F::TILE, wave, lane);
    }
    // the rows' statistics, by waves that bring rows too: the wait for a stage counts loads, LOADS or more of them per stage
    const auto bring = [&](int which) {
      const int r = r0 + lane;
      const float* src = which ? (r < a.M ? a.delta + (long long)pr * a.M + r : (const float*)attn_zero)
                               : (r < a.M ? a.lse2 + (long long)pr * a.M + r : &attn_inf);
      dma4(src, base + F::stats_at + buf * 512 + which * 256);
    };
    if constexpr (RB > Dm::RPI) {
      if (wave < 2 && lane < RB) bring(wave);
    } else if (wave == 0 && lane < RB) {
      bring(0), bring(1);
    }
  };

  for (int half = 0; half < (a.causal ? 2 : 1); ++half) {
    const int tile = half ? a.tiles - 1 - tu : tu;
    if (half && tile <= tu) break;
    if (half) __syncthreads();  // the join of the first tile has been read
    if (half == 0 || WR > 1) {  // (the join has been here)
      clear_tail<T, DP>(attn_smem, F::NBUF * 2 * RB, a.D, F::NTH);
      if (VL) clear_tail<T, DP>(attn_smem + F::v_at, BN, a.D, F::NTH);
    }
    const int j0 = tile * BN, key = j0 + wn * TM + n;
    const bool seen = key < p.len && (!km || km[key]);
    // first row that sees the lane's key / the wave's first key / all of the wave's keys
    const int rmin = first_row(key), rany = first_row(j0 + wn * TM), rall = first_row(j0 + wn * TM + TM - 1);
    int rbeg = j0 < p.len ? first_row(j0) : INT_MAX, rend;
    if (rbeg < a.M) {
      const int b0 = rbeg / RB, blocks = (a.M + RB - 1) / RB - b0;
      rbeg = (b0 + (int)((long long)blocks * split / a.nsplit)) * RB;
      rend = min((b0 + (int)((long long)blocks * (split + 1) / a.nsplit)) * RB, a.M);
    } else {
      rbeg = rend = 0;  // no row sees a key of the tile
    }

    typename M::Frag kf[KF], vf[VL ? 1 : KF];
    load_frags<T, KF>(kf, seen ? (const T*)a.k + p.b * a.sk.b + key * a.sk.l + p.hk * a.sk.h : nullptr, a.D, h);
    if constexpr (VL) {
      Dma<T, DP, BN, NW>::rows(
          [&](int j) {
            return j0 + j < p.len && (!km || km[j0 + j]) ? (const T*)a.v + p.b * a.sv.b + (j0 + j) * a.sv.l + p.hk * a.sv.h
                                                         : (const T*)nullptr;
          },
          a.D, base + F::v_at, wave, lane);
    } else {
      load_frags<T, KF>(vf, seen ? (const T*)a.v + p.b * a.sv.b + key * a.sv.l + p.hk * a.sv.h : nullptr, a.D, h);
    }

    typename M::Acc dk[MD], dv[MD];
#pragma unroll
    for (int md = 0; md < MD; ++md) dk[md] = dv[md] = (typename M::Acc)(0.f);
    if (rbeg < rend) request(rbeg, 0);
    if (F::NBUF == 3 && rbeg + RB < rend) request(rbeg + RB, 1);
    settle(kf);
    if (!VL) settle(vf);
    stage_done<0, true>();
    int buf = 0;
    for (int r0 = rbeg; r0 < rend; r0 += RB) {
      const bool more = r0 + (F::NBUF - 1) * RB < rend;
      if (more) request(r0 + (F::NBUF - 1) * RB, F::NBUF == 2 ? buf ^ 1 : buf == 0 ? 2 : buf - 1);
      const int rw = r0 + wr * F::RW;
      if (rw + F::RW > rany) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int lr = wr * F::RW + mt * TM;  // the tile's row in the stage
          const char* qt = attn_smem + buf * F::STAGE + lr * L::ROWB;
          const char* dt = qt + F::TILE;
          typename M::Acc sc = (typename M::Acc)(0.f), dp = (typename M::Acc)(0.f);
          if (sizeof(T) == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int f = 0; f < KF; ++f) {
            sc = M::mma(L::rowfrag(qt, f, lane), kf[f], sc);
            if constexpr (VL) dp = M::mma(L::rowfrag(dt, f, lane), L::rowfrag(vw, f, lane), dp);
            else dp = M::mma(L::rowfrag(dt, f, lane), vf[f], dp);
          }
          __builtin_amdgcn_s_setprio(0);
          if (rw < rall) {  // some rows do not see some keys: a score of -inf leaves a probability of zero
            const int from = rmin - rw - mt * TM - 4 * h;
#pragma unroll
            for (int x = 0; x < M::NC; ++x)
              if (M::crow(x, 0) < from) sc[x] = -INFINITY;
          }
          const float* st = stats + buf * 128 + lr;
#pragma unroll
          for (int q = 0; q < M::NC / 4; ++q) {
            const int r = M::crow(4 * q, h);
            const fl4 l4 = *(const fl4*)(st + r), d4 = *(const fl4*)(st + 64 + r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = exp2_(__builtin_fmaf(sc[4 * q + e], a.c, -l4[e]));
              sc[4 * q + e] = x;
              dp[4 * q + e] = x * (dp[4 * q + e] - d4[e]);
            }
          }
#pragma unroll
          for (int t = 0; t < TM / 16; ++t) {
            const typename M::Frag pf = M::pack(sc, t), sf = M::pack(dp, t);
#pragma unroll
            for (int md = 0; md < MD; ++md) {
              dv[md] = M::mma(L::colfrag(dt + 16 * t * L::ROWB, md, lane), pf, dv[md]);
              dk[md] = M::mma(L::colfrag(qt + 16 * t * L::ROWB, md, lane), sf, dk[md]);
            }
          }
        }
      }
      // the next stage has landed; the one after it may be on its way
      if (F::NBUF == 3 && more) stage_done<F::LOADS, true>();
      else stage_done<0, true>();
      buf = buf == F::NBUF - 1 ? 0 : buf + 1;
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

// ------------------------------------------------------------------------------------- gradients of short sequences at once
// Up to MB rows and MB keys (the samples of a ray): one workgroup holds the problem, reads it once and forms all five products;
// the two kernels above would read it twice and take seven.  Every wave owns TM keys, walks the rows for its dk and dv, and
// leaves ds in LDS by keys; then it owns TM rows and reads ds back by columns for dq.  128 rows go in two halves, so that ds
// takes half the room and more workgroups share a CU; two waves then share a tile's dq, each with every other tile of keys.
// Bound by the chain of its phases (loads, five products, a barrier, stores) at 4 to 8 waves per SIMD: 1024 rays of 64 masked samples,
// 4 fp32 heads of 16: 45 us, 3.0 TB/s of its own bytes; 4096 x 128 in bf16: 205 us, 2.6 TB/s (one piece instead of halves: 290).
template <typename T, int DP, int MB>
struct Short {
  using L = Lay<T, DP>;
  static constexpr int HALVES = MB == 128 ? 2 : 1, HR = MB / HALVES;
  using X = Lay<T, HR>;
  static constexpr int TM = Mt<T>::TM, NW = MB / TM, NTH = 64 * NW, TILE = MB * L::ROWB;
  static constexpr int q_at = 0, do_at = TILE, k_at = 2 * TILE, x_at = 3 * TILE, st_at = x_at + MB * X::ROWB, dq_at = st_at + 2 * MB * 4;
  static constexpr size_t lds = dq_at + (HALVES - 1) * NW / 2 * L::MD * Mt<T>::NC * 64 * 4;
  static constexpr bool fits = lds <= 128 * 1024;
};

template <typename T, int DP, int MB>
__global__ void __launch_bounds__(64 * MB / Mt<T>::TM, 2) k_attn_short(const AttnP a) {
  using F = Short<T, DP, MB>;
  using M = Mt<T>;
  using L = typename F::L;
  using X = typename F::X;
  constexpr int TM = M::TM, NW = F::NW, KF = L::KF, MD = L::MD;
  int pr, unit;
  if (!locate(a.B * a.Hkv, 1, pr, unit)) return;
  const Prob p = problem(a, pr);
  const int lane = threadIdx.x & 63, wave = wave_index(), n = lane & (TM - 1), h = lane / TM;
  clear_tail<T, DP>(attn_smem, 3 * MB, a.D, F::NTH);
  const unsigned base = lds_address(attn_smem);
  const unsigned char* km = a.key_mask ? a.key_mask + p.b * a.mask_sb : nullptr;
  // which keys are there; the first row and key of the problem, from which 32-bit offsets reach all others
  constexpr int WORDS = (MB + 63) / 64;
  unsigned long long bits[WORDS];
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int j = 64 * w + lane;
    bits[w] = __ballot(j < p.len && (!km || km[j]));
  }
  const auto there = [&](int j) { return (bool)(bits[WORDS == 1 ? 0 : j >> 6] >> (j & 63) & 1); };
  const T* q0 = (const T*)a.q + p.b * a.sq.b + (long long)p.hk * a.G * a.sq.h;
  const T* d0 = (const T*)a.dout + p.b * a.sdo.b + (long long)p.hk * a.G * a.sdo.h;
  const T* k0 = (const T*)a.k + p.b * a.sk.b + p.hk * a.sk.h;
  const T* v0 = (const T*)a.v + p.b * a.sv.b + p.hk * a.sv.h;
  const long long o0 = ((long long)p.b * a.Lq * a.Hq + p.hk * a.G) * a.D;  // of the problem's first row in out and dq
  const auto off = [&](int r, int sl, int sh) {
    const int i = row_pos(a, r);
    return i * sl + (r - i * a.G) * sh;
  };
  using Dm = Dma<T, DP, MB, NW>;
  if (a.G == 1 && a.M == MB) {
    Dm::whole(q0, a.sq.l, a.D, base + F::q_at, wave, lane);
    Dm::whole(d0, a.sdo.l, a.D, base + F::do_at, wave, lane);
  } else {
    const auto in = [&](int r) { return r < a.M; };
    Dm::near(q0, [&](int r) { return off(min(r, a.M - 1), (int)a.sq.l, (int)a.sq.h); }, in, a.D, base + F::q_at, wave, lane);
    Dm::near(d0, [&](int r) { return off(min(r, a.M - 1), (int)a.sdo.l, (int)a.sdo.h); }, in, a.D, base + F::do_at, wave, lane);
  }
  bool all = MB >= 64;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) all &= bits[w] == ~0ull;
  if (all) Dm::whole(k0, a.sk.l, a.D, base + F::k_at, wave, lane);
  else Dm::near(k0, [&](int j) { return j * (int)a.sk.l; }, there, a.D, base + F::k_at, wave, lane);

  // the wave's keys
  const int key = wave * TM + n;
  const bool seen = there(key);
  typename M::Frag kf[KF], vf[KF];
  load_frags_near<T, KF>(kf, k0, key * (int)a.sk.l, seen, a.D, h);
  load_frags_near<T, KF>(vf, v0, key * (int)a.sv.l, seen, a.D, h);
  // the wave's rows: log-sum-exp (powers of two; +inf: no probability) and do.o
  const int row = wave * TM + n;
  const bool live = row < a.M;
  float* st = (float*)(attn_smem + F::st_at);  // [MB] log-sum-exp, [MB] delta
  {
    const int rr = live ? row : 0, i = row_pos(a, rr);
    typename M::Frag of[KF], df[KF];
    load_frags_near<T, KF>(of, (const T*)a.out + o0, off(rr, a.Hq * a.D, a.D), live, a.D, h);
    load_frags_near<T, KF>(df, d0, off(rr, (int)a.sdo.l, (int)a.sdo.h), live, a.D, h);
    float delta = 0.f;
#pragma unroll
    for (int f = 0; f < KF; ++f)
#pragma unroll
      for (int e = 0; e < M::EP; ++e) delta = __builtin_fmaf((float)df[f][e], (float)of[f][e], delta);
    delta = col_sum<T>(delta);
    const float* l0 = a.lse + ((long long)p.b * a.Hq + p.hk * a.G) * a.Lq;
    float lse2 = live ? l0[(unsigned)((rr - i * a.G) * a.Lq + i)] * LOG2E : INFINITY;
    if (lse2 == -INFINITY) lse2 = INFINITY;
    if (h == 0) st[row] = lse2, st[MB + row] = delta;
  }
  const auto first_row = [&](int j) { return !a.causal || j <= p.qs ? 0 : j - p.qs >= a.Lq ? INT_MAX : (j - p.qs) * a.G; };
  const int rmin = first_row(key), rany = first_row(wave * TM), rall = first_row(wave * TM + TM - 1);
  stage_done<0, true>();

  const int ktiles = (p.len + TM - 1) / TM;
  char* xs = attn_smem + F::x_at;
  const int xp = X::phys(key), xw = X::swz(xp);
  typename M::Acc dk[MD], dv[MD];
#pragma unroll
  for (int md = 0; md < MD; ++md) dk[md] = dv[md] = (typename M::Acc)(0.f);
  // one tile of rows: its part of dv and dk, and ds -> LDS (columns from x0 on).  `partly`: some of the tile's rows do not see
  // some of the keys.
  const auto rows = [&](int r0, int x0, auto partly) {
    const char* qt = attn_smem + F::q_at + r0 * L::ROWB;
    const char* dt = attn_smem + F::do_at + r0 * L::ROWB;
    typename M::Acc sc = (typename M::Acc)(0.f), dp = (typename M::Acc)(0.f);
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      sc = M::mma(L::rowfrag(qt, f, lane), kf[f], sc);
      dp = M::mma(L::rowfrag(dt, f, lane), vf[f], dp);
    }
#pragma unroll
    for (int q = 0; q < M::NC / 4; ++q) {
      const int r = r0 + M::crow(4 * q, h);
      const fl4 l4 = *(const fl4*)(st + r), d4 = *(const fl4*)(st + MB + r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = exp2_(__builtin_fmaf(sc[4 * q + e], a.c, -l4[e]));
        if (decltype(partly)::value && (r + e < rmin || !seen)) x = 0.f;
        sc[4 * q + e] = x;
        dp[4 * q + e] = x * (dp[4 * q + e] - d4[e]);
      }
    }
#pragma unroll
    for (int t = 0; t < TM / 16; ++t) {
      const typename M::Frag pf = M::pack(sc, t), sf = M::pack(dp, t);
#pragma unroll
      for (int md = 0; md < MD; ++md) {
        dv[md] = M::mma(L::colfrag(dt + 16 * t * L::ROWB, md, lane), pf, dv[md]);
        dk[md] = M::mma(L::colfrag(qt + 16 * t * L::ROWB, md, lane), sf, dk[md]);
      }
      typedef T V4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int g = 0; g < M::EP / 4; ++g) {  // four neighbouring rows of the lane's key
        V4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = sf[4 * g + e];
        const int at = (r0 - x0 + M::crow(M::EP * t + 4 * g, h)) * (int)sizeof(T);
        *(V4*)(xs + xp * X::ROWB + ((at >> 4 ^ xw) << 4) + (at & 15)) = y;
      }
    }
  };
  const bool hidden = __any(!seen);
  for (int half = 0; half < F::HALVES; ++half) {
    const int x0 = half * F::HR, x1 = min(x0 + F::HR, a.M);
    if (wave < ktiles) {
      int r0 = x0;
      for (; r0 < x1 && r0 + TM <= rany; r0 += TM) {  // rows before the first that sees a key of the wave: ds is zero
#pragma unroll
        for (int x = 0; x < TM * TM * (int)sizeof(T) / 1024; ++x) {
          const int px = X::phys(wave * TM + lane % TM), at = (r0 - x0) * (int)sizeof(T) + ((lane / TM) + x * (64 / TM)) * 16;
          *(u4v*)(xs + px * X::ROWB + ((at >> 4 ^ X::swz(px)) << 4)) = u4v{0, 0, 0, 0};
        }
      }
      for (; r0 < x1 && (hidden || r0 < rall); r0 += TM) rows(r0, x0, std::true_type());
      for (; r0 < x1; r0 += TM) rows(r0, x0, std::false_type());
    }
    if (half == F::HALVES - 1 && key < a.Lk) {
      if (!seen) {  // a hidden key's gradients are zero: its probabilities are, but not their products with what overflowed
#pragma unroll
        for (int md = 0; md < MD; ++md) dk[md] = dv[md] = (typename M::Acc)(0.f);
      }
      const long long g0 = ((long long)p.b * a.Lk * a.Hkv + p.hk) * a.D;
      const unsigned at = (unsigned)(key * a.Hkv * a.D);
      store_cols<T, T, MD>(dk, a.scale, (T*)a.dk + g0 + at, a.D, h);
      store_cols<T, T, MD>(dv, 1.f, (T*)a.dv + g0 + at, a.D, h);
    }
    __syncthreads();
    constexpr int TW = NW / F::HALVES;  // tiles of rows of a half
    const int tile = wave % TW, part = wave / TW, q0 = x0 + tile * TM;
    typename M::Acc dq[MD];
#pragma unroll
    for (int md = 0; md < MD; ++md) dq[md] = (typename M::Acc)(0.f);
    if (q0 < a.M) {
      for (int kt = part; kt < ktiles; kt += F::HALVES) {
#pragma unroll
        for (int t = 0; t < TM / 16; ++t) {
          const int j = kt * TM + 16 * t;
          const typename M::Frag sf = X::colfrag(xs + j * X::ROWB, tile, lane);
#pragma unroll
          for (int md = 0; md < MD; ++md) dq[md] = M::mma(L::colfrag(attn_smem + F::k_at + j * L::ROWB, md, lane), sf, dq[md]);
        }
      }
    }
    if constexpr (F::HALVES == 2) {
      fl4* x = (fl4*)(attn_smem + F::dq_at) + tile * MD * (M::NC / 4) * 64 + lane;
      if (part) {
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
          for (int q = 0; q < M::NC / 4; ++q) {
            fl4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = dq[md][4 * q + e];
            x[(md * (M::NC / 4) + q) * 64] = y;
          }
      }
      __syncthreads();
      if (!part) {
#pragma unroll
        for (int md = 0; md < MD; ++md)
#pragma unroll
          for (int q = 0; q < M::NC / 4; ++q) {
            const fl4 y = x[(md * (M::NC / 4) + q) * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) dq[md][4 * q + e] += y[e];
          }
      }
    }
    const int qr = q0 + n;
    if (part == 0 && qr < a.M) store_cols<T, T, MD>(dq, a.scale, (T*)a.dq + o0 + (unsigned)off(qr, a.Hq * a.D, a.D), a.D, h);
  }
}

// ------------------------------------------------------------------------------------------------------------ host
template <typename K>
int launch(K kernel, const char* name, long long grid, int threads, size_t lds, hipStream_t st, const AttnP& a) {
  GPN_REQUIRE(grid * threads < (1ll << 32), "%s: %lld workgroups of %d", name, grid, threads);
  if (grid == 0) return GPN_OK;
  if (lds > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return gpn_set_error(GPN_E_LAUNCH, "hipFuncSetAttribute(%zu B LDS): %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, a);
  GPN_LAUNCH_CHECK(name);
  return GPN_OK;
}

// Two waves along the rows and two along the keys instead of four along the rows: twice as many workgroups of half the rows,
// where one workgroup of the latter per CU takes all tiles, or two where tiles differ or heads are narrow: they fill the card and
// even out.  (2048 causal positions, 8 heads: fp32 of 64, forward 84 -> 59 us, backward 214 -> 175; bf16 of 128, forward 45 -> 36.
// 2 x 2000 causal, 8 fp32 heads of 32: 77 -> 49, 206 -> 160.)  With more, keys are read more often than that gains (3 x 1000, 16
// heads of 128: 40 against 47, 131 against 140).
bool is_mid(long long prob, long long M, bool f32, int D, bool causal) {
  const long long large = prob * ((M + (f32 ? 63 : 127)) / (f32 ? 64 : 128));
  return large <= (causal || D <= 64 ? 512 : 256);
}

// How a forward call is cut: rows per workgroup, keys per stage, splits of the keys.
struct Plan {
  bool one_piece;  // few enough keys for one workgroup's registers
  bool few;        // one tile of rows per workgroup, whose waves divide the keys
  bool mid;        // two waves along the rows, two along the keys
  int bm, tiles, nsplit, split_keys;
};

Plan plan_forward(const gpn_attn_args_t* x) {
  Plan p = {};
  const bool f32 = x->dtype == GPN_DT_F32;
  const long long M = (long long)x->Lq * (x->Hq / x->Hkv), prob = (long long)x->B * x->Hkv;
  const int big = f32 ? 64 : 128, small = f32 ? 16 : 32;
  p.nsplit = 1, p.split_keys = x->Lk;
  p.one_piece = x->Lk <= (f32 && x->D > 64 ? 64 : 128);  // 64 KB of keys and values: two workgroups per CU
  if (p.one_piece) {  // as many waves as there are tiles of rows, four at most
    p.bm = M <= small ? small : M <= 2 * small ? 2 * small : 4 * small;
    p.tiles = (int)((M + p.bm - 1) / p.bm);
    return p;
  }
  // Tiles of few rows also for narrow heads under `causal` whose tiles see anything from nothing to all keys and fill no more than
  // the card: the finest cut evens out best (3000 positions, 8 query and 2 key/value heads of 64: 29 against 38 us; 2048, 8 heads:
  // 21 against 28).  Fewer positions fill the card only where there are enough problems for larger tiles (4 x 1024, 8 heads: 23
  // against 19).
  const long long large = prob * ((M + big - 1) / big);
  const bool steep = x->causal && !f32 && x->D <= 64 && x->Lq >= x->Lk / 2 && large <= (x->Lk >= 2048 ? 256 : 128) &&
                     prob * ((M + small - 1) / small) >= 256;
  p.few = M <= small || steep;
  // wide fp32 heads, of which such a wave takes 16 keys at a time: only where tiles of many rows leave no room for parts of the keys
  // (3 x 333, 6 query and 3 key/value heads, 1021 keys: of 80 40 against 43 us, of 128 54 against 58)
  p.mid = !p.few && is_mid(prob, M, f32, x->D, x->causal) && !(f32 && x->D > 64 && large <= 128);
  p.bm = p.few ? small : p.mid ? big / 2 : big;
  p.tiles = (int)((M + p.bm - 1) / p.bm);
  // The card takes 512 workgroups (two per CU).  Where there are half as many or fewer the keys are cut too, into parts of
  // min_part or more so that a part outweighs its share of the join.  (One query, 8 heads, 64 K keys: 64 parts 51 us, 5.3 TB/s;
  // twice as many workgroups for eight queries of uneven lengths 82 against 76 us.)  Workgroups of many rows that are more than
  // half the CUs' number only where the keys are long or their products slow (1100 queries, 16 K keys, 8 heads of 128: 240 us in
  // one part, 130 in three; fp32 2 x 400, 8 query and 4 key/value heads of 128, 1400 keys: 132 and 70; but 2 x 777, 8 query and 2
  // key/value heads of 64: 16, 21).
  const long long units = prob * p.tiles, min_part = f32 ? 128 : 256;
  const long long split_to = M <= small ? 512 : steep ? 0 : (f32 && x->D > 64) || x->Lk >= 2048 ? 256 : 128;
  const long long s = units < 1 || units > split_to ? 1 : std::min({512 / units, x->Lk / min_part, (long long)MAX_SPLIT});
  if (s > 1) {
    p.split_keys = (int)(((x->Lk + s - 1) / s + 63) / 64 * 64);
    p.nsplit = (x->Lk + p.split_keys - 1) / p.split_keys;
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
  GPN_REQUIRE(x->scale >= 1e-30f && x->scale <= 1e30f, "%s: scale must be between 1e-30 and 1e30", name);
  return GPN_OK;
}

// Strides of batches, positions and heads; nothing lies a stride away along a dimension of one, so that stride counts as 0,
// whatever a slice of a larger tensor has there.
Strides strides(const long long* s, int B, int L, int H) { return Strides{B > 1 ? s[0] : 0, L > 1 ? s[1] : 0, H > 1 ? s[2] : 0}; }
Strides query_strides(const gpn_attn_args_t* x, const long long* s) { return strides(s, x->B, x->Lq, x->Hq); }
Strides key_strides(const gpn_attn_args_t* x, const long long* s) { return strides(s, x->B, x->Lk, x->Hkv); }

int check_tensor(const void* p, int size, const char* what, const char* name, Strides s = {}) {
  GPN_REQUIRE(p, "%s: null %s", name, what);
  GPN_REQUIRE(((size_t)p & 15) == 0, "%s: %s is not 16-byte aligned", name, what);
  for (const long long x : {s.b, s.l, s.h})
    GPN_REQUIRE(x >= 0 && x * size % 16 == 0, "%s: stride %lld of %s is not a multiple of 16 bytes", name, x, what);
  return GPN_OK;
}

AttnP fill(const gpn_attn_args_t* x) {
  AttnP a = {};
  a.q = x->q, a.k = x->k, a.v = x->v, a.dout = x->dout;
  a.out = x->out, a.dq = x->dq, a.dk = x->dk, a.dv = x->dv;
  a.sq = query_strides(x, x->q_stride), a.sdo = query_strides(x, x->dout_stride);
  a.sk = key_strides(x, x->k_stride), a.sv = key_strides(x, x->v_stride);
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
  if (pl.one_piece) {
    constexpr int TM = Mt<T>::TM;
#define GPN_ONE(NW, KB) \
  launch(k_attn_one_piece<T, DP, NW, KB>, "k_attn_one_piece", grid, 64 * NW, OnePiece<T, DP, NW, KB>::lds, st, a)
    if (a.Lk <= 64) return pl.bm == TM ? GPN_ONE(1, 64) : pl.bm == 2 * TM ? GPN_ONE(2, 64) : GPN_ONE(4, 64);
    if constexpr (!F32 || DP <= 64) return pl.bm == TM ? GPN_ONE(1, 128) : pl.bm == 2 * TM ? GPN_ONE(2, 128) : GPN_ONE(4, 128);
#undef GPN_ONE
  }
  if (pl.few) {
    constexpr int KT = F32 && DP > 64 ? 16 : 32, WK = 16 * KT * Lay<T, DP>::ROWB > 64 * 1024 ? 2 : 4;  // two workgroups per CU
    using F = Few<T, DP, WK, KT>;
    rc = launch(k_attn_few<T, DP, WK, KT>, "k_attn_few", grid, F::NTH, F::lds, st, a);
  } else {
    constexpr int KT = F32 && DP > 64 ? 32 : 64;  // two stages of 64 KB at most: two workgroups per CU
    if (pl.mid) {
      using F = Fwd<T, DP, 2, KT>;
      constexpr size_t join = 2 * (F::L::MD * Mt<T>::NC + 2) * 64 * 4;
      rc = launch(k_attn_fwd<T, DP, 2, 2, KT>, "k_attn_fwd", grid, 256, std::max((size_t)F::lds, join), st, a);
    } else {
      using F = Fwd<T, DP, 4, KT>;
      rc = launch(k_attn_fwd<T, DP, 4, 1, KT>, "k_attn_fwd", grid, F::NTH, F::lds, st, a);
    }
  }
  if (rc || pl.nsplit == 1) return rc;
  const long long rows = (long long)a.B * a.Hkv * a.M;
  return launch(k_attn_join<T>, "k_attn_join", (rows + 7) / 8, 256, 0, st, a);
}

// Keys of a workgroup of the dk / dv kernel: 4 waves' tiles.
int dkv_keys(bool f32) { return f32 ? 64 : 128; }

// Parts that the rows of a key tile are cut into: one round of workgroups (one per CU; two for heads whose sums leave room), with
// 256 rows or more each, so that a part's products outweigh its sums' way through memory.  (2 x 4096 causal, 4 key/value heads
// of 128: 598 us with one round, 614 with two.)
int plan_dkv(const gpn_attn_args_t* x) {
  const long long M = (long long)x->Lq * (x->Hq / x->Hkv);
  const int bn = dkv_keys(x->dtype == GPN_DT_F32);
  long long tiles = (x->Lk + bn - 1) / bn;
  if (x->causal) tiles = (tiles + 1) / 2;
  const long long units = (long long)x->B * x->Hkv * tiles;
  const long long slots = x->D > 32 ? 256 : 512;
  if (units == 0 || units > slots / 2) return 1;
  long long s = slots / units;
  if (s > M / 256) s = M / 256;
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

template <typename T, int DP, int MB>
int short_t(const AttnP& a, hipStream_t st) {
  using F = Short<T, DP, MB>;
  if constexpr (F::fits) return launch(k_attn_short<T, DP, MB>, "k_attn_short", grid_of((long long)a.B * a.Hkv, 1), F::NTH, F::lds, st, a);
  return gpn_set_error(GPN_E_ARG, "gpn_attn_backward: no such kernel");
}

// Strides that 128 rows times them, and their groups, stay far within 32 bits.
bool is_near(const gpn_attn_args_t* x) {
  const long long m = 1 << 20;
  bool near = (long long)x->Hq * x->D < m;
  for (const Strides& s : {query_strides(x, x->q_stride), query_strides(x, x->dout_stride), key_strides(x, x->k_stride),
                           key_strides(x, x->v_stride)})
    near &= s.l < m && s.h < m;
  return near;
}

// A problem that one workgroup's LDS holds with its ds: 128 rows and keys, at most this wide.
bool is_short(const gpn_attn_args_t* x) {
  const long long n = std::max((long long)x->Lq * (x->Hq / x->Hkv), (long long)x->Lk);
  return n >= 1 && n <= 128 && x->D <= (x->dtype == GPN_DT_BF16 || n <= 64 ? 64 : 32) && is_near(x);
}

template <typename T, int DP, int WR>
int dkv_t(const AttnP& a, long long grid, hipStream_t st) {
  using F = Dkv<T, DP, 4, WR>;
  static_assert(F::BN == (sizeof(T) == 4 ? 64 : 128) && F::lds <= 160 * 1024, "dkv_keys, LDS");
  return launch(k_attn_dkv<T, DP, 4, WR>, "k_attn_dkv", grid, F::NTH, F::lds, st, a);
}

template <typename T, int DP>
int backward_t(AttnP& a, bool shrt, int nsplit, hipStream_t st) {
  constexpr bool F32 = sizeof(T) == 4;
  const long long prob = (long long)a.B * a.Hkv;
  if constexpr (DP <= 64) {
    if (shrt) {
      const int n = std::max(a.M, a.Lk);
      return n <= 32 ? short_t<T, DP, 32>(a, st) : n <= 64 ? short_t<T, DP, 64>(a, st) : short_t<T, DP, 128>(a, st);
    }
  }
  int rc;
  {
    constexpr int KT = F32 && DP > 64 ? 32 : 64;
    if (is_mid(prob, a.M, F32, a.D, a.causal)) {
      using F = Fwd<T, DP, 2, KT>;
      constexpr size_t join = (size_t)2 * F::L::MD * Mt<T>::NC * 64 * 4;
      a.tiles = (a.M + F::BM - 1) / F::BM;
      rc = launch(k_attn_dq<T, DP, 2, KT, 2>, "k_attn_dq", grid_of(prob, a.tiles), 256, std::max((size_t)F::lds, join), st, a);
    } else {
      using F = Fwd<T, DP, 4, KT>;
      a.tiles = (a.M + F::BM - 1) / F::BM;
      rc = launch(k_attn_dq<T, DP, 4, KT, 1>, "k_attn_dq", grid_of(prob, a.tiles), 256, F::lds, st, a);
    }
    if (rc) return rc;
  }
  a.tiles = (a.Lk + dkv_keys(F32) - 1) / dkv_keys(F32), a.nsplit = nsplit;
  const long long units = (long long)(a.causal ? (a.tiles + 1) / 2 : a.tiles) * nsplit, grid = grid_of(prob, units);
  // Pairs of waves per key tile keep the parts few where there are few tiles; with two workgroups for every CU in any case,
  // workgroups of four waves wait for each other less (4 x 4096 of 16 heads of 64: 1107 us for the backward in pairs, 1062).
  if (!F32 && prob * units >= 512) rc = dkv_t<T, DP, F32 ? 2 : 1>(a, grid, st);
  else rc = dkv_t<T, DP, 2>(a, grid, st);
  if (rc || nsplit == 1) return rc;
  return launch(k_attn_dkv_join<T>, "k_attn_dkv_join", ((long long)a.B * a.Lk * a.Hkv * a.D / 2 + 255) / 256, 256, 0, st, a);
}

// Head widths are padded with zeros to the next of these.  fp32 has two more, multiples of its 16-wide tiles: its products are what
// takes the time (2 x 800, 8 heads of 48, forward and backward: 34 + 99 us, as 64 wide 40 + 121; 64 x 60 rows and keys of 80: 15 + 49,
// as 96 16 + 54).
template <typename Fn>
int by_width(bool f32, int D, Fn fn) {
#define GPN_WIDTH(T, DP) \
  if (D <= DP) return fn(T(), std::integral_constant<int, DP>())
  if (f32) {
    GPN_WIDTH(float, 16);
    GPN_WIDTH(float, 32);
    GPN_WIDTH(float, 48);
    GPN_WIDTH(float, 64);
    GPN_WIDTH(float, 80);
    GPN_WIDTH(float, 96);
    GPN_WIDTH(float, 128);
  }
  GPN_WIDTH(bf16, 16);
  GPN_WIDTH(bf16, 32);
  GPN_WIDTH(bf16, 64);
  GPN_WIDTH(bf16, 96);
  GPN_WIDTH(bf16, 128);
#undef GPN_WIDTH
  return gpn_set_error(GPN_E_ARG, "no kernel for heads of %d", D);
}

}  // namespace

extern "C" size_t gpn_attn_workspace_bytes(const gpn_attn_args_t* x, int backward) {
  if (check_args(x, "gpn_attn_workspace_bytes") || x->B == 0 || x->Lq == 0) return 0;
  const size_t rows = (size_t)x->B * x->Hq * x->Lq;
  if (backward && is_short(x)) return 0;
  if (backward) {  // delta, log-sum-exp in powers of two, and the parts of dk and dv
    const int s = plan_dkv(x);
    return 2 * align256(rows * 4) + (s > 1 ? (size_t)s * 2 * x->B * x->Lk * x->Hkv * x->D * 4 : 0);
  }
  const Plan p = plan_forward(x);
  return p.nsplit == 1 ? 0 : align256(rows * p.nsplit * 4) + rows * p.nsplit * x->D * 4;
}

extern "C" int gpn_attn_forward(const gpn_attn_args_t* x, gpn_stream_t stream) {
  const char* name = "gpn_attn_forward";
  if (int rc = check_args(x, name)) return rc;
  if (x->B == 0 || x->Lq == 0) return GPN_OK;
  const int size = x->dtype == GPN_DT_F32 ? 4 : 2;
  if (int rc = check_tensor(x->q, size, "q", name, query_strides(x, x->q_stride))) return rc;
  if (x->Lk > 0) {
    if (int rc = check_tensor(x->k, size, "k", name, key_strides(x, x->k_stride))) return rc;
    if (int rc = check_tensor(x->v, size, "v", name, key_strides(x, x->v_stride))) return rc;
  }
  if (int rc = check_tensor(x->out, size, "out", name)) return rc;
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
  return by_width(x->dtype == GPN_DT_F32, x->D,
                  [&](auto t, auto dp) { return forward_t<decltype(t), decltype(dp)::value>(a, pl, st); });
}

extern "C" int gpn_attn_backward(const gpn_attn_args_t* x, gpn_stream_t stream) {
  const char* name = "gpn_attn_backward";
  if (int rc = check_args(x, name)) return rc;
  if (x->B == 0 || (x->Lq == 0 && x->Lk == 0)) return GPN_OK;
  const int size = x->dtype == GPN_DT_F32 ? 4 : 2;
  if (x->Lq > 0) {
    if (int rc = check_tensor(x->q, size, "q", name, query_strides(x, x->q_stride))) return rc;
    if (int rc = check_tensor(x->dout, size, "dout", name, query_strides(x, x->dout_stride))) return rc;
    if (int rc = check_tensor(x->out, size, "out", name)) return rc;
    if (int rc = check_tensor(x->dq, size, "dq", name)) return rc;
    GPN_REQUIRE(x->lse, "%s: null lse", name);
  }
  if (x->Lk > 0) {
    if (int rc = check_tensor(x->k, size, "k", name, key_strides(x, x->k_stride))) return rc;
    if (int rc = check_tensor(x->v, size, "v", name, key_strides(x, x->v_stride))) return rc;
    if (int rc = check_tensor(x->dk, size, "dk", name)) return rc;
    if (int rc = check_tensor(x->dv, size, "dv", name)) return rc;
  }
  const size_t need = gpn_attn_workspace_bytes(x, 1);
  GPN_REQUIRE(x->workspace_bytes >= need && (need == 0 || x->workspace), "%s: workspace of %zu bytes, %zu needed", name,
              x->workspace_bytes, need);
  AttnP a = fill(x);
  const bool shrt = is_short(x);
  const int nsplit = shrt ? 1 : plan_dkv(x);
  a.delta = (float*)x->workspace;
  const size_t stat = align256((size_t)x->B * x->Hq * x->Lq * 4);
  a.lse2 = (float*)((char*)x->workspace + stat);
  a.part_o = (float*)((char*)x->workspace + 2 * stat);
  hipStream_t st = (hipStream_t)stream;
  return by_width(x->dtype == GPN_DT_F32, x->D,
                  [&](auto t, auto dp) { return backward_t<decltype(t), decltype(dp)::value>(a, shrt, nsplit, st); });
}
