// Differential attention, backward (diff_attn.hpp: formula, fragment layout, tile search).
//
// With P_i the two softmax maps, W = P1 - lam P2 and D_i = rowsum(dO o (P_i V)):
//   dV = W^T dO,  dP = dO V^T,  dS1 = P1 o (dP - D1),  dS2 = -lam P2 o (dP - D2),
//   dQ_i = s dS_i K_i,  dK_i = s dS_i^T Q_i,  dlam = -sum D2.
// P_i is recomputed from the saved log-sum-exp.  k_diff_delta forms D; k_diff_bwd has workgroups that own keys and walk the
// queries and workgroups that own queries and walk the keys (the scores and dP twice, but no atomics: every sum in one fixed order).
//
// Two graphs of 4,175 and 5,261 nodes, 8 heads over 4 of 64 columns, bf16: 1.04 ms in a replayed graph = 620 TFLOP/s of its 28 d flops per
// pair and head (20 d with the scores and dP once), 1.17 under a tracer, as the figures below were taken.  No unit is saturated: LDS 42 % busy (every fragment that a wavefront reads there serves one 16 x 16
// tile), vector units 40 %, matrix units 27 %; 213 registers leave two wavefronts per SIMD, which wait for each other's phases.
// Tried and slower: two tiles per wavefront (373 registers, one wavefront per SIMD: 1.51 ms; for dQ alone, spilling: 1.44), three
// wavefronts per SIMD (28 registers spilled: 1.29), eight wavefronts per workgroup (half the staging: 1.18-1.22), a copy of the step
// without the mask's selects (1.16, and 90 against 86 us in fp32).
#include "diff_attn.hpp"

namespace diffattn {
namespace {

// dS in two 16-bit terms.  With one, the error of dQ and dK is 1.41 to 1.5 times that of a gradient that is rounded once at its end, and
// more (up to 1.9) where heads are narrow and rows see few keys: the terms of a sum cancel and their errors do not.  Up to 32
// columns, where both second products of dS are small, it is kept in two: 1.0 to 1.1 times, for 39.8 us instead of 38.6 for a whole pass
// over 32 trees of ~123 nodes and 523 instead of 487 over 9 causal graphs of 2,108 (4 heads over 1, 16 columns).  Above that in one: the
// backward of two graphs of ~4,700 nodes, 64 columns, would take 1,165 us instead of 1,060.
template <typename T, int DQ>
constexpr bool two_terms() { return sizeof(T) == 2 && DQ == 32; }

// float16 holds nothing below 2^-25, and W and dS are that small in long rows or under small output gradients (which are what a loss
// without a scale gives).  So a column of tiles (a key in dkv, a query in dq) keeps its dS times 2^up, a power of two that starts at
// kUpStart and falls, accumulators with it, where a dS would pass 2^15; W <= 1 + |lam| has a power of its own.  All of that is exact, and
// taken out at the end.  Segments of 600 and 130 rows, 24 columns, output gradients of 1e-4: dq and dk 0.0018 and 0.0012 off, which is
// what rounding them to float16 costs; 0.0068 and 0.0081 without.  Whole backward of two graphs of ~4,700 nodes, 64 columns, float16:
// 1,120 us against 1,080; ordered sequences of ~2,600, 128 columns: 1,135 against 1,180.
template <typename T>
constexpr bool ranged() { return false; }
template <>
constexpr bool ranged<f16>() { return true; }
constexpr int kUpStart = 13;
constexpr float kMost = 0x1p15f;

// powers of two that bring the largest magnitude `m` of a column (the same in its four lanes) to 2^12; 0 where it is fine or not finite
__device__ __forceinline__ int lower_by(float m) { return m > kMost && m < kInf ? (int)(__float_as_uint(m) >> 23) - 127 - 12 : 0; }
__device__ __forceinline__ float largest(float x, const f32x4& v) {
#pragma unroll
  for (int r = 0; r < 4; ++r) x = fmaxf(x, fabsf(v[r]));
  return x;
}

constexpr int kDeltaRows = 64;   // rows of one k_diff_delta workgroup

// D2 = dO . O2 and D1 = dO . O + lam D2: sixteen lanes per (row, head), sixteen rows of a head at a time.  HBM-bound: 9,436 rows of 8 heads
// of 128 columns, bf16 with what O lost and fp32 O2: 97 MB in 16 us.
template <typename T>
__global__ __launch_bounds__(256) void k_diff_delta(Args a, float* __restrict__ delta) {
  const int h = blockIdx.y, lane = threadIdx.x & 15, dv = 2 * a.d;
  const float lam = load_lam(a, h, static_cast<const T*>(nullptr));
#pragma unroll
  for (int it = 0; it < kDeltaRows / 16; ++it) {
    const int64_t r = (int64_t)blockIdx.x * kDeltaRows + it * 16 + (threadIdx.x >> 4);
    float x = 0.f, y = 0.f;
    if (r < a.Nq && a.lse[(int64_t)h * a.Nq + r] < kInf) {   // a row that saw no key has no gradient, whatever dO holds there
      const T* dop = static_cast<const T*>(a.dout) + r * a.do_rs + h * a.do_hs;
      const T* op = static_cast<const T*>(a.o) + (r * a.H + h) * dv;
      const T* restp = static_cast<const T*>(a.o_rest) + (r * a.H + h) * dv;
      const float* o2p = a.o2 + (r * a.H + h) * dv;
      for (int c = lane * 4; c < dv; c += 64) {
        const vec_t<T, 4> go = *reinterpret_cast<const vec_t<T, 4>*>(dop + c), o = *reinterpret_cast<const vec_t<T, 4>*>(op + c);
        const f32x4 o2 = *reinterpret_cast<const f32x4*>(o2p + c);
        vec_t<T, 4> rest = vec_t<T, 4>(0);
        if (sizeof(T) == 2 && a.o_rest) rest = *reinterpret_cast<const vec_t<T, 4>*>(restp + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x += (float)go[i] * ((float)o[i] + (float)rest[i]);
          y += (float)go[i] * o2[i];
        }
      }
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) {
      x += __shfl_xor(x, o);
      y += __shfl_xor(y, o);
    }
    if (lane == 0 && r < a.Nq) {
      delta[(int64_t)h * a.Nq + r] = x + lam * y;
      delta[((int64_t)a.H + h) * a.Nq + r] = y;
    }
  }
}

// dlam of one head from the partial sums that dq() left
template <typename T>
__global__ __launch_bounds__(256) void k_diff_dlam(const float* __restrict__ part, int64_t n, void* __restrict__ out, int f32) {
  __shared__ double sh[4];
  const int h = blockIdx.x;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += (double)part[h * n + i];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = -(sh[0] + sh[1] + sh[2] + sh[3]);
  if (f32 || sizeof(T) == 4)
    static_cast<float*>(out)[h] = (float)s;
  else
    static_cast<T*>(out)[h] = (T)(float)s;
}

// dK, dV: a wavefront owns KT x 16 keys (column of every tile) of one key head, its K and V rows in registers; the workgroup walks
// the queries of each head of the group in blocks of 32 rows of Q (both maps) and dO, two blocks in LDS.  Each fragment read from
// LDS serves KT tiles; W and dS go into the second products from the registers they are computed in.
template <typename T, int DQ, int KT, bool Masked>
__device__ __forceinline__ void dkv(const Args& a, const float* __restrict__ delta, int tile, int hk, unsigned char* lds_raw) {
  constexpr int DV = 2 * DQ, ST = DQ / 32, SV = DV / 32, DQT = DQ / 16, DVT = DV / 16, BQ = 32;
  typedef Tl<T, DV> L;
  T* tiles = reinterpret_cast<T*>(lds_raw);                              // [2][Q | dO]
  float* lst_all = reinterpret_cast<float*>(tiles + 4 * BQ * DV);        // [2][lse1 | lse2 | D1 | D2]

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
  const int bm = (blockDim.x >> 6) * 16 * KT, group = a.H / a.Hk, dv = 2 * a.d;
  const Tile t = find_tile(a.k_ptr, a.B, a.Nk, bm, tile);
  if (t.rows <= 0) return;
  int q0 = 0, nq = 0;
  if (t.seg < a.B) {
    q0 = clamp_row(a.q_ptr[t.seg], a.Nq);
    nq = max(0, clamp_row(a.q_ptr[t.seg + 1], a.Nq) - q0);
  }
  const int shift = t.len - nq;                                       // query i sees keys <= i + shift
  const int first = a.causal ? max(0, t.local - shift) : 0;           // first query that sees a key of this tile

  const RowShare<BQ> share;
  const Stager<T, BQ, DV, 2> stage_q(a.q_rs, a.q_ms, a.d);
  const Stager<T, BQ, DV, 1> stage_o(a.do_rs, 0, dv);
  // block of 32 queries from qb of head h -> tiles and statistics `buf`; rows past the segment repeat its last one, `cut` below
  // leaves them out
  auto fetch = [&](int h, int qb, int buf) __attribute__((always_inline)) {
    T* lq = tiles + buf * 2 * BQ * DV;
    float* lst = lst_all + buf * 4 * BQ;
    const int64_t base = (int64_t)q0 + qb;
    const int n = min(BQ, nq - qb);
    for (int i = wave; i < 2; i += (int)(blockDim.x >> 6)) {   // lse1 | lse2, then D1 | D2: one load of 64 lanes each
      const float* src = (i ? delta : (const float*)a.lse) + ((int64_t)(lane >> 5) * a.H + h) * a.Nq + base + min(lane & 31, n - 1);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                       (__attribute__((address_space(3))) void*)(lst + i * 64), 4, 0, 0);
    }
    const T* qs = static_cast<const T*>(a.q) + base * a.q_rs + h * a.q_hs;
    const T* os = static_cast<const T*>(a.dout) + base * a.do_rs + h * a.do_hs;
    stage_q(lq, qs, a.q_rs, a.q_ms, n, a.d);
    stage_o(lq + BQ * DV, os, a.do_rs, 0, n, dv);
  };
  if (first < nq) fetch(hk * group, first, 0);

  Frag<T> kf[2][KT][ST], vf[KT][SV];
  int64_t row[KT];
  bool live[KT];
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    const int r = (wave * KT + i) * 16 + col;
    row[i] = r < t.rows ? (int64_t)t.first + r : -1;
    live[i] = row[i] >= 0 && (!Masked || a.keep[row[i]]);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        kf[m][i][s] = frag_zero<T>();
        if (live[i] && s * 32 + g * 8 < a.d)
          kf[m][i][s] = frag_load(static_cast<const T*>(a.k) + row[i] * a.k_rs + hk * a.k_hs + m * a.k_ms + s * 32 + g * 8);
      }
#pragma unroll
    for (int s = 0; s < SV; ++s) {
      vf[i][s] = frag_zero<T>();
      if (live[i] && s * 32 + g * 8 < dv)
        vf[i][s] = frag_load(static_cast<const T*>(a.v) + row[i] * a.v_rs + hk * a.v_hs + s * 32 + g * 8);
    }
  }
  f32x4 gk[2][KT][DQT], gv[KT][DVT];
#pragma unroll
  for (int i = 0; i < KT; ++i) {
#pragma unroll
    for (int c = 0; c < DQT; ++c) gk[0][i][c] = gk[1][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DVT; ++c) gv[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale2 = a.scale * kLog2e;
  int up[KT], up_w = kUpStart;   // of dS, of W (float16)
  float w_up[KT];                // 2^(up_w - up): what P is times 2^up lacks for W
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    up[i] = kUpStart;
    w_up[i] = 1.f;
  }
  int buf = 0;
  for (int h = hk * group; h < hk * group + group && first < nq; ++h) {
   const float lam = load_lam(a, h, static_cast<const T*>(nullptr));
   if constexpr (ranged<T>()) {
     const int most = 14 + 127 - (int)(__float_as_uint(1.f + fabsf(lam)) >> 23);   // 2^most (1 + |lam|) < 2^15
     if (up_w > most) {
       const float f = __builtin_amdgcn_ldexpf(1.f, most - up_w);
       up_w = most;
#pragma unroll
       for (int i = 0; i < KT; ++i) {
         w_up[i] *= f;
#pragma unroll
         for (int c = 0; c < DVT; ++c) gv[i][c] *= f;
       }
     }
   }
   for (int qb = first; qb < nq; qb += BQ, buf ^= 1) {
    tiles_ready();
    if constexpr (Masked) {   // a query that sees no key has weights of 0 and may hold anything
      T* t0 = tiles + buf * 2 * BQ * DV;
      if (!(lst_all[buf * 4 * BQ + share.row] < kInf)) {
        share.template zero<T, DV>(t0);
        share.template zero<T, DV>(t0 + BQ * DV);
      }
      __syncthreads();
    }
    if (qb + BQ < nq)
      fetch(h, qb + BQ, buf ^ 1);
    else if (h + 1 < hk * group + group)
      fetch(h + 1, first, buf ^ 1);
    const bool cut = Masked || a.causal || qb + BQ > nq;   // (uniform)
    const T* lq = tiles + buf * 2 * BQ * DV;
    const T* lo = lq + BQ * DV;
    const float* lst = lst_all + buf * 4 * BQ;

    f32x4 s[2][KT][2], dp[KT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < KT; ++i) s[0][i][u] = s[1][i][u] = dp[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const Frag<T> qf = L::frag(lq, u * 16 + col, m * DQ + st * 32 + g * 8);
#pragma unroll
          for (int i = 0; i < KT; ++i) s[m][i][u] = mma(qf, kf[m][i][st], s[m][i][u]);
        }
#pragma unroll
      for (int st = 0; st < SV; ++st) {
        const Frag<T> of = L::frag(lo, u * 16 + col, st * 32 + g * 8);
#pragma unroll
        for (int i = 0; i < KT; ++i) dp[i][u] = mma(of, vf[i][st], dp[i][u]);
      }
      const f32x4 l1 = *reinterpret_cast<const f32x4*>(lst + u * 16 + g * 4), l2 = *reinterpret_cast<const f32x4*>(lst + BQ + u * 16 + g * 4);
      const f32x4 d1 = *reinterpret_cast<const f32x4*>(lst + 2 * BQ + u * 16 + g * 4), d2 = *reinterpret_cast<const f32x4*>(lst + 3 * BQ + u * 16 + g * 4);
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const int key = t.local + (wave * KT + i) * 16 + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i][u][r], scale2, ranged<T>() ? (float)up[i] - l1[r] : -l1[r]));
          float p2 = lam * __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][i][u][r], scale2, ranged<T>() ? (float)up[i] - l2[r] : -l2[r]));
          if (cut) {
            const int q = qb + u * 16 + g * 4 + r;
            const bool in = live[i] && q < nq && (!a.causal || key <= q + shift);
            p1 = in ? p1 : 0.f;
            p2 = in ? p2 : 0.f;
            if (Masked) dp[i][u][r] = in ? dp[i][u][r] : 0.f;
          }
          const float x = dp[i][u][r];
          dp[i][u][r] = ranged<T>() ? (p1 - p2) * w_up[i] : p1 - p2;   // W
          s[0][i][u][r] = p1 * (x - d1[r]);      // dS1
          s[1][i][u][r] = p2 * (d2[r] - x);      // dS2
        }
      }
    }
    if constexpr (ranged<T>()) {
      float m[KT];
      bool past = false;
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        m[i] = largest(largest(largest(largest(0.f, s[0][i][0]), s[0][i][1]), s[1][i][0]), s[1][i][1]);
        past |= m[i] > kMost;
      }
      if (__any(past)) {
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          const int by = lower_by(over_groups(m[i], [](float x, float y) { return fmaxf(x, y); }));
          const float f = __builtin_amdgcn_ldexpf(1.f, -by);
          up[i] -= by;
          w_up[i] = __builtin_amdgcn_ldexpf(w_up[i], by);
#pragma unroll
          for (int c = 0; c < DQT; ++c) {
            gk[0][i][c] *= f;
            gk[1][i][c] *= f;
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[0][i][u] *= f;
            s[1][i][u] *= f;
          }
        }
      }
    }
    Frag<T> w[KT], ds[2][KT], lost[2][KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      w[i] = frag_pack<T>(dp[i][0], dp[i][1]);
      ds[0][i] = frag_pack<T>(s[0][i][0], s[0][i][1]);
      ds[1][i] = frag_pack<T>(s[1][i][0], s[1][i][1]);
      if constexpr (two_terms<T, DQ>()) {
        lost[0][i] = frag_lost(s[0][i][0], s[0][i][1], ds[0][i]);
        lost[1][i] = frag_lost(s[1][i][0], s[1][i][1], ds[1][i]);
      }
    }
#pragma unroll
    for (int c = 0; c < DVT; ++c) {
      const Frag<T> of = L::frag_tr(lo, 0, c * 16, lane);
#pragma unroll
      for (int i = 0; i < KT; ++i) gv[i][c] = mma(of, w[i], gv[i][c]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const Frag<T> qf = L::frag_tr(lq, 0, m * DQ + c * 16, lane);
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          gk[m][i][c] = mma(qf, ds[m][i], gk[m][i][c]);
          if constexpr (two_terms<T, DQ>()) gk[m][i][c] = mma(qf, lost[m][i], gk[m][i][c]);
        }
      }
   }
  }
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    if (row[i] < 0) continue;
    const float down = ranged<T>() ? __builtin_amdgcn_ldexpf(1.f, -up[i]) : 1.f, down_w = ranged<T>() ? __builtin_amdgcn_ldexpf(1.f, -up_w) : 1.f;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const int x = c * 16 + g * 4;
        if (x < a.d) store4(static_cast<T*>(a.dk) + row[i] * a.dk_rs + hk * a.dk_hs + m * a.dk_ms + x, live[i] ? gk[m][i][c] * (a.scale * down) : f32x4{0.f, 0.f, 0.f, 0.f});
      }
#pragma unroll
    for (int c = 0; c < DVT; ++c) {
      const int x = c * 16 + g * 4;
      if (x < dv) store4(static_cast<T*>(a.dv) + row[i] * a.dv_rs + hk * a.dv_hs + x, live[i] ? gv[i][c] * down_w : f32x4{0.f, 0.f, 0.f, 0.f});
    }
  }
}

// dQ: a wavefront owns QT x 16 queries (column of every tile) of one head, its Q and dO rows in registers; the workgroup walks the
// keys in blocks of 32 rows of K (both maps) and V, two blocks in LDS.  On the way it sums P2 o dP, unrounded: dlam = -sum D2 cancels
// over all rows and columns, and dO . O2 of weights that were rounded to 16 bits would show.
template <typename T, int DQ, int QT, bool Masked>
__device__ __forceinline__ void dq(const Args& a, const float* __restrict__ delta, float* __restrict__ part, int tile, int h,
                                   unsigned char* lds_raw) {
  constexpr int DV = 2 * DQ, ST = DQ / 32, SV = DV / 32, DQT = DQ / 16, BK = 32;
  typedef Tl<T, DV> L;
  T* tiles = reinterpret_cast<T*>(lds_raw);                              // [2][K | V]
  int* lkeep = reinterpret_cast<int*>(tiles + 4 * BK * DV);              // [2][BK]

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
  const int bm = (blockDim.x >> 6) * 16 * QT, hk = h / (a.H / a.Hk), dv = 2 * a.d;
  const Tile t = find_tile(a.q_ptr, a.B, a.Nq, bm, tile);
  float* lsum = reinterpret_cast<float*>(reinterpret_cast<int*>(tiles + 4 * BK * DV) + 2 * BK);   // [wavefronts]
  if (t.rows <= 0) {
    if (threadIdx.x == 0) *part = 0.f;
    return;
  }
  int k0 = 0, nk = 0;
  if (t.seg < a.B) {
    k0 = clamp_row(a.k_ptr[t.seg], a.Nk);
    nk = max(0, clamp_row(a.k_ptr[t.seg + 1], a.Nk) - k0);
  }
  const int shift = nk - t.len;
  const int last = a.causal ? min(nk, max(0, t.local + t.rows + shift)) : nk;
  const float lam = load_lam(a, h, static_cast<const T*>(nullptr)), scale2 = a.scale * kLog2e;

  const RowShare<BK> share;
  bool kept = true;   // whether this thread's row of the block that was fetched last is a key
  const Stager<T, BK, DV, 2> stage_k(a.k_rs, a.k_ms, a.d);
  const Stager<T, BK, DV, 1> stage_v(a.v_rs, 0, dv);
  auto fetch = [&](int kb, int buf) __attribute__((always_inline)) {
    T* lk = tiles + buf * 2 * BK * DV;
    const int64_t base = (int64_t)k0 + kb;
    const int n = min(BK, nk - kb);
    const T* ks = static_cast<const T*>(a.k) + base * a.k_rs + hk * a.k_hs;
    const T* vs = static_cast<const T*>(a.v) + base * a.v_rs + hk * a.v_hs;
    if constexpr (Masked) kept = share.row < n && a.keep[base + min(share.row, n - 1)];
    stage_k(lk, ks, a.k_rs, a.k_ms, n, a.d);
    stage_v(lk + BK * DV, vs, a.v_rs, 0, n, dv);
  };
  if (last > 0) fetch(0, 0);

  Frag<T> qf[2][QT][ST], of[QT][SV];
  int64_t row[QT];
  int seen[QT];
  float lse[2][QT], dl[2][QT];   // lse less `up`
  int up[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = (wave * QT + i) * 16 + col;
    row[i] = r < t.rows ? (int64_t)t.first + r : -1;
    seen[i] = a.causal ? t.local + r + shift + 1 : nk;
    up[i] = kUpStart;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int64_t at = ((int64_t)m * a.H + h) * a.Nq + row[i];
      lse[m][i] = row[i] >= 0 ? (ranged<T>() ? a.lse[at] - (float)kUpStart : a.lse[at]) : kInf;
      dl[m][i] = row[i] >= 0 ? delta[at] : 0.f;
    }
    const bool ok = lse[0][i] < kInf;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        qf[m][i][s] = frag_zero<T>();
        if (ok && s * 32 + g * 8 < a.d)
          qf[m][i][s] = frag_load(static_cast<const T*>(a.q) + row[i] * a.q_rs + h * a.q_hs + m * a.q_ms + s * 32 + g * 8);
      }
#pragma unroll
    for (int s = 0; s < SV; ++s) {
      of[i][s] = frag_zero<T>();
      if (ok && s * 32 + g * 8 < dv)
        of[i][s] = frag_load(static_cast<const T*>(a.dout) + row[i] * a.do_rs + h * a.do_hs + s * 32 + g * 8);
    }
  }
  const int all_see = a.causal ? t.local + wave * QT * 16 + shift + 1 : nk;
  float d2[QT] = {};   // times 2^up
  f32x4 gq[2][QT][DQT];
#pragma unroll
  for (int i = 0; i < QT; ++i)
#pragma unroll
    for (int c = 0; c < DQT; ++c) gq[0][i][c] = gq[1][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};

  int buf = 0;
  for (int kb = 0; kb < last; kb += BK, buf ^= 1) {
    tiles_ready();
    const T* lk = tiles + buf * 2 * BK * DV;
    const T* lv = lk + BK * DV;
    if constexpr (Masked) {   // scores and dP of dropped keys are cut below; their rows of K would meet a dS of 0
      if (!kept) share.template zero<T, DV>(const_cast<T*>(lk));
      if (share.part == 0) lkeep[buf * BK + share.row] = kept;
      __syncthreads();
    }
    if (kb + BK < last) fetch(kb + BK, buf ^ 1);
    const bool cut = Masked || kb + BK > all_see;   // (uniform over the wavefront)

    f32x4 s[2][QT][2], dp[QT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < QT; ++i) s[0][i][u] = s[1][i][u] = dp[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const Frag<T> kf = L::frag(lk, u * 16 + col, m * DQ + st * 32 + g * 8);
#pragma unroll
          for (int i = 0; i < QT; ++i) s[m][i][u] = mma(kf, qf[m][i][st], s[m][i][u]);
        }
#pragma unroll
      for (int st = 0; st < SV; ++st) {
        const Frag<T> vf = L::frag(lv, u * 16 + col, st * 32 + g * 8);
#pragma unroll
        for (int i = 0; i < QT; ++i) dp[i][u] = mma(vf, of[i][st], dp[i][u]);
      }
      int4 kp = make_int4(1, 1, 1, 1);
      if constexpr (Masked) kp = *reinterpret_cast<const int4*>(lkeep + buf * BK + u * 16 + g * 4);
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i][u][r], scale2, -lse[0][i]));
          float p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][i][u][r], scale2, -lse[1][i]));
          if (cut) {
            const bool in = (&kp.x)[r] && kb + u * 16 + g * 4 + r < seen[i];
            p1 = in ? p1 : 0.f;
            p2 = in ? p2 : 0.f;
            if (Masked) dp[i][u][r] = in ? dp[i][u][r] : 0.f;
          }
          d2[i] = __builtin_fmaf(p2, dp[i][u][r], d2[i]);
          s[0][i][u][r] = p1 * (dp[i][u][r] - dl[0][i]);
          s[1][i][u][r] = p2 * (dl[1][i] - dp[i][u][r]);
        }
    }
    if constexpr (ranged<T>()) {
      float m[QT];
      bool past = false;
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        m[i] = largest(largest(largest(largest(0.f, s[0][i][0]), s[0][i][1]), s[1][i][0]), s[1][i][1]);
        past |= m[i] > kMost;
      }
      if (__any(past)) {
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          const int by = lower_by(over_groups(m[i], [](float x, float y) { return fmaxf(x, y); }));
          const float f = __builtin_amdgcn_ldexpf(1.f, -by);
          up[i] -= by;
          lse[0][i] += (float)by;
          lse[1][i] += (float)by;
          d2[i] *= f;
#pragma unroll
          for (int c = 0; c < DQT; ++c) {
            gq[0][i][c] *= f;
            gq[1][i][c] *= f;
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[0][i][u] *= f;
            s[1][i][u] *= f;
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      Frag<T> ds[QT], lost[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        ds[i] = frag_pack<T>(s[m][i][0], s[m][i][1]);
        if constexpr (two_terms<T, DQ>()) lost[i] = frag_lost(s[m][i][0], s[m][i][1], ds[i]);
      }
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const Frag<T> kf = L::frag_tr(lk, 0, m * DQ + c * 16, lane);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          gq[m][i][c] = mma(kf, ds[i], gq[m][i][c]);
          if constexpr (two_terms<T, DQ>()) gq[m][i][c] = mma(kf, lost[i], gq[m][i][c]);
        }
      }
    }
  }
  float d2_all = 0.f;
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const float down = ranged<T>() ? __builtin_amdgcn_ldexpf(1.f, -up[i]) : 1.f;
    d2_all += d2[i] * down;
    if (row[i] < 0) continue;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const int x = c * 16 + g * 4;
        if (x < a.d) store4(static_cast<T*>(a.dq) + row[i] * a.dq_rs + h * a.dq_hs + m * a.dq_ms + x, gq[m][i][c] * ((m ? a.scale * lam : a.scale) * down));
      }
  }
  for (int o = 32; o; o >>= 1) d2_all += __shfl_xor(d2_all, o);
  if (lane == 0) lsum[wave] = d2_all;
  __syncthreads();
  if (threadIdx.x == 0) {
    d2_all = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) d2_all += lsum[w];
    *part = d2_all;
  }
}

// Both in one launch: the workgroups of dK / dV first (they are the longest), then those of dQ, which fill the CUs that the last
// uneven round of the first kind leaves idle.
template <typename T, int DQ, int RT, bool Masked>
__global__ __launch_bounds__(256, DQ == 32 ? 3 : sizeof(T) == 2 && DQ == 64 ? 2 : 1) void k_diff_bwd(Args a, const float* __restrict__ delta, float* __restrict__ part,
                                                                    int k_tiles, int q_tiles) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds_raw[];
  const int k_units = xcd_grid(k_tiles * a.Hk), b = blockIdx.x;
  if (b < k_units) {
    const Unit u = xcd_unit(b, k_tiles, a.Hk);
    if (u.tile < k_tiles && u.head < a.Hk) dkv<T, DQ, RT, Masked>(a, delta, u.tile, u.head, lds_raw);
  } else {
    const Unit u = xcd_unit(b - k_units, q_tiles, a.H);
    if (u.tile < q_tiles && u.head < a.H) dq<T, DQ, RT, Masked>(a, delta, part + u.head * q_tiles + u.tile, u.tile, u.head, lds_raw);
  }
}

// Registers (and with them wavefronts per SIMD): 32 columns hold 137 in 16 bits and, spilling 12, 168 in fp32, three either way; 64 columns
// 213 in 16 bits (two); the rest one.
template <typename T, int DQ, int RT>
int launch_bwd(const Args& a, float* part, hipStream_t s) {
  constexpr int per_wave = 16 * RT;
  const int longest = a.max_q > a.max_k ? a.max_q : a.max_k;
  const bool known = a.max_q > 0 && a.max_k > 0;
  // as in the forward: no idle wavefronts where all segments are short
  const int waves = known && longest <= per_wave ? 1 : known && longest <= 2 * per_wave ? 2 : 4, bm = waves * per_wave;
  const int k_tiles = a.Nk > 0 ? (int)(a.Nk / bm) + a.B + 1 : 0, q_tiles = a.Nq > 0 ? (int)(a.Nq / bm) + a.B + 1 : 0;
  const unsigned grid = (unsigned)(xcd_grid(k_tiles * a.Hk) + xcd_grid(q_tiles * a.H));
  const size_t lds = 2 * 32 * (4 * DQ * sizeof(T) + 4 * sizeof(float)) + 16;
  if (grid == 0) return 0;
  if (a.keep)
    k_diff_bwd<T, DQ, RT, true><<<grid, waves * 64, lds, s>>>(a, a.ws, part, k_tiles, q_tiles);
  else
    k_diff_bwd<T, DQ, RT, false><<<grid, waves * 64, lds, s>>>(a, a.ws, part, k_tiles, q_tiles);
  return q_tiles;
}

}  // namespace

// ws: delta [2, H, Nq] | partial sums of dlam [H, tiles of queries]
template <typename T>
void backward(const Args& a, hipStream_t s) {
  float* part = a.ws + (int64_t)2 * a.H * a.Nq;
  if (a.Nq > 0) k_diff_delta<T><<<dim3((unsigned)((a.Nq + kDeltaRows - 1) / kDeltaRows), (unsigned)a.H), 256, 0, s>>>(a, a.ws);
  const int parts = a.d <= 32 ? launch_bwd<T, 32, 1>(a, part, s) : a.d <= 64 ? launch_bwd<T, 64, 1>(a, part, s) : launch_bwd<T, 128, 1>(a, part, s);
  k_diff_dlam<T><<<(unsigned)a.H, 256, 0, s>>>(part, parts, a.dlam, a.lam_f32);
}

template void backward<float>(const Args&, hipStream_t);
template void backward<bf16>(const Args&, hipStream_t);
template void backward<f16>(const Args&, hipStream_t);

}  // namespace diffattn

extern "C" size_t gps_diff_attn_bwd_workspace_floats(int64_t Nq, int H, int B) {
  if (Nq < 0 || H <= 0 || B < 0) return 0;
  return (size_t)H * (2 * (size_t)Nq + (size_t)Nq / 16 + B + 1);   // tiles of 16 rows at least
}
