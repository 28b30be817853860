// Differential attention, backward (diff_attn.hpp: formula, fragment layout, tile search).
//
// With P_i the two softmax maps, W = P1 - lam P2 and D_i = rowsum(dO o (P_i V)):
//   dV = W^T dO,  dP = dO V^T,  dS1 = P1 o (dP - D1),  dS2 = -lam P2 o (dP - D2),
//   dQ_i = s dS_i K_i,  dK_i = s dS_i^T Q_i,  dlam = -sum D2.
// P_i is recomputed from the saved log-sum-exp.  k_diff_delta forms D and dlam's partial sums; k_diff_dkv owns keys and walks the
// queries, k_diff_dq owns queries and walks the keys: no atomics, every sum in one fixed order.
#include "diff_attn.hpp"

namespace diffattn {
namespace {

constexpr int kDeltaRows = 64;   // rows of one k_diff_delta workgroup

// D2 = dO . O2 and D1 = dO . O + lam D2, one wavefront per (row, head); the workgroup's sum of D2 is one term of -dlam
template <typename T>
__global__ __launch_bounds__(256) void k_diff_delta(Args a, float* __restrict__ delta, float* __restrict__ part) {
  __shared__ float sh[4];
  const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dv = 2 * a.d;
  const float lam = load_lam(a, h, static_cast<const T*>(nullptr));
  const int64_t r0 = (int64_t)blockIdx.x * kDeltaRows;
  float total = 0.f;
  for (int j = wave; j < kDeltaRows; j += 4) {
    const int64_t r = r0 + j;
    if (r >= a.Nq) break;
    float x = 0.f, y = 0.f;
    if (a.lse[(int64_t)h * a.Nq + r] < kInf) {   // a row that saw no key has no gradient, whatever dO holds there
      const T* dop = static_cast<const T*>(a.dout) + r * a.do_rs + h * a.do_hs;
      const T* op = static_cast<const T*>(a.o) + (r * a.H + h) * dv;
      const float* o2p = a.o2 + (r * a.H + h) * dv;
      for (int c = lane; c < dv; c += 64) {
        const float go = (float)dop[c];
        x += go * (float)op[c];
        y += go * o2p[c];
      }
    }
    for (int o = 32; o; o >>= 1) {
      x += __shfl_xor(x, o);
      y += __shfl_xor(y, o);
    }
    if (lane == 0) {
      delta[(int64_t)h * a.Nq + r] = x + lam * y;
      delta[((int64_t)a.H + h) * a.Nq + r] = y;
    }
    total += y;
  }
  if (lane == 0) sh[wave] = total;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)h * gridDim.x + blockIdx.x] = sh[0] + sh[1] + sh[2] + sh[3];
}

template <typename T>
__global__ __launch_bounds__(64) void k_diff_dlam(const float* __restrict__ part, int64_t n, void* __restrict__ out, int f32) {
  const int h = blockIdx.x;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 64) s += (double)part[h * n + i];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if (threadIdx.x == 0) {
    if (f32 || sizeof(T) == 4)
      static_cast<float*>(out)[h] = (float)-s;
    else
      static_cast<T*>(out)[h] = (T)(float)-s;
  }
}

template <typename T>
struct BCfg {
  static constexpr int Pad = 16 / sizeof(T);
};

// dK, dV: a wavefront owns KT x 16 keys (column of every tile) of one key head; the workgroup walks the queries of each head of
// the group in blocks of 32 rows of Q (both maps) and dO staged in LDS
template <typename T, int DQ, int KT>
__global__ __launch_bounds__(256) void k_diff_dkv(Args a, const float* __restrict__ delta) {
  constexpr int DV = 2 * DQ, ST = DQ / 32, SV = DV / 32, DQT = DQ / 16, DVT = DV / 16, BQ = 32;
  constexpr int LQ = 2 * DQ + BCfg<T>::Pad, LO = DV + BCfg<T>::Pad;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  T* lq = reinterpret_cast<T*>(lds_raw);
  T* lo = lq + BQ * LQ;
  float* lst = reinterpret_cast<float*>(lo + BQ * LO);   // lse1 | lse2 | D1 | D2 of the block's rows

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
  const int bm = (blockDim.x >> 6) * 16 * KT, hk = blockIdx.y, group = a.H / a.Hk, dv = 2 * a.d;
  const Tile t = find_tile(a.k_ptr, a.B, a.Nk, bm, blockIdx.x);
  if (t.rows <= 0) return;
  int q0 = 0, nq = 0;
  if (t.seg < a.B) {
    q0 = clamp_row(a.q_ptr[t.seg], a.Nq);
    nq = max(0, clamp_row(a.q_ptr[t.seg + 1], a.Nq) - q0);
  }
  const int shift = t.len - nq;                                       // query i sees keys <= i + shift
  const int first = a.causal ? max(0, t.local - shift) / BQ * BQ : 0;  // first block that sees a key of this tile

  Frag<T> kf[2][KT][ST], vf[KT][SV];
  int64_t row[KT];
  bool live[KT];
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    const int r = (wave * KT + i) * 16 + col;
    row[i] = r < t.rows ? (int64_t)t.first + r : -1;
    live[i] = row[i] >= 0 && (!a.keep || a.keep[row[i]]);
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

  for (int hg = 0; hg < group; ++hg) {
    const int h = hk * group + hg;
    const float lam = load_lam(a, h, static_cast<const T*>(nullptr));
    for (int qb = first; qb < nq; qb += BQ) {
      const int64_t base = (int64_t)q0 + qb;
      const int n = min(BQ, nq - qb);
      const float* lse = a.lse + (int64_t)h * a.Nq + base;
      auto any = [&](int r) { return lse[r] < kInf; };
      __syncthreads();
#pragma unroll
      for (int m = 0; m < 2; ++m)
        stage<T, BQ, DQ>(lq + m * DQ, LQ, static_cast<const T*>(a.q) + base * a.q_rs + h * a.q_hs + m * a.q_ms, a.q_rs, n, a.d, any);
      stage<T, BQ, DV>(lo, LO, static_cast<const T*>(a.dout) + base * a.do_rs + h * a.do_hs, a.do_rs, n, dv, any);
      for (int i = threadIdx.x; i < 4 * BQ; i += blockDim.x) {
        const int which = i / BQ, r = i % BQ;
        const float* src = (which < 2 ? (const float*)a.lse : delta) + ((int64_t)(which & 1) * a.H + h) * a.Nq + base;
        lst[i] = r < n ? src[r] : (which < 2 ? kInf : 0.f);
      }
      __syncthreads();

      f32x4 s[2][KT][2], dp[KT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < KT; ++i) s[0][i][u] = s[1][i][u] = dp[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int st = 0; st < ST; ++st) {
            const Frag<T> qf = frag_load(lq + (u * 16 + col) * LQ + m * DQ + st * 32 + g * 8);
#pragma unroll
            for (int i = 0; i < KT; ++i) s[m][i][u] = mma(qf, kf[m][i][st], s[m][i][u]);
          }
#pragma unroll
        for (int st = 0; st < SV; ++st) {
          const Frag<T> of = frag_load(lo + (u * 16 + col) * LO + st * 32 + g * 8);
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
            const bool in = live[i] && (!a.causal || key <= qb + u * 16 + g * 4 + r + shift);
            const float p1 = in ? __builtin_amdgcn_exp2f(s[0][i][u][r] * scale2 - l1[r]) : 0.f;
            const float p2 = in ? lam * __builtin_amdgcn_exp2f(s[1][i][u][r] * scale2 - l2[r]) : 0.f;
            const float x = dp[i][u][r];
            dp[i][u][r] = p1 - p2;                 // W
            s[0][i][u][r] = p1 * (x - d1[r]);      // dS1
            s[1][i][u][r] = -p2 * (x - d2[r]);     // dS2
          }
        }
      }
      Frag<T> w[KT], ds[2][KT];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        w[i] = frag_pack<T>(dp[i][0], dp[i][1]);
        ds[0][i] = frag_pack<T>(s[0][i][0], s[0][i][1]);
        ds[1][i] = frag_pack<T>(s[1][i][0], s[1][i][1]);
      }
#pragma unroll
      for (int c = 0; c < DVT; ++c) {
        const Frag<T> of = frag_tr(lo, LO, 0, c * 16, lane);
#pragma unroll
        for (int i = 0; i < KT; ++i) gv[i][c] = mma(of, w[i], gv[i][c]);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < DQT; ++c) {
          const Frag<T> qf = frag_tr(lq, LQ, 0, m * DQ + c * 16, lane);
#pragma unroll
          for (int i = 0; i < KT; ++i) gk[m][i][c] = mma(qf, ds[m][i], gk[m][i][c]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    if (row[i] < 0) continue;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const int x = c * 16 + g * 4;
        if (x < a.d) store4(static_cast<T*>(a.dk) + row[i] * a.dk_rs + hk * a.dk_hs + m * a.dk_ms + x, gk[m][i][c] * a.scale);
      }
#pragma unroll
    for (int c = 0; c < DVT; ++c) {
      const int x = c * 16 + g * 4;
      if (x < dv) store4(static_cast<T*>(a.dv) + row[i] * a.dv_rs + hk * a.dv_hs + x, gv[i][c]);
    }
  }
}

// dQ: a wavefront owns QT x 16 queries (column of every tile) of one head; the workgroup walks the keys in blocks of 32 rows of K
// (both maps) and V staged in LDS
template <typename T, int DQ, int QT>
__global__ __launch_bounds__(256) void k_diff_dq(Args a, const float* __restrict__ delta) {
  constexpr int DV = 2 * DQ, ST = DQ / 32, SV = DV / 32, DQT = DQ / 16, BK = 32;
  constexpr int LK = 2 * DQ + BCfg<T>::Pad, LV = DV + BCfg<T>::Pad;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  T* lk = reinterpret_cast<T*>(lds_raw);
  T* lv = lk + BK * LK;
  int* lkeep = reinterpret_cast<int*>(lv + BK * LV);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
  const int bm = (blockDim.x >> 6) * 16 * QT, h = blockIdx.y, hk = h / (a.H / a.Hk), dv = 2 * a.d;
  const Tile t = find_tile(a.q_ptr, a.B, a.Nq, bm, blockIdx.x);
  if (t.rows <= 0) return;
  int k0 = 0, nk = 0;
  if (t.seg < a.B) {
    k0 = clamp_row(a.k_ptr[t.seg], a.Nk);
    nk = max(0, clamp_row(a.k_ptr[t.seg + 1], a.Nk) - k0);
  }
  const int shift = nk - t.len;
  const int last = a.causal ? min(nk, max(0, t.local + t.rows + shift)) : nk;
  const float lam = load_lam(a, h, static_cast<const T*>(nullptr)), scale2 = a.scale * kLog2e;

  Frag<T> qf[2][QT][ST], of[QT][SV];
  int64_t row[QT];
  int seen[QT];
  float lse[2][QT], dl[2][QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = (wave * QT + i) * 16 + col;
    row[i] = r < t.rows ? (int64_t)t.first + r : -1;
    seen[i] = a.causal ? t.local + r + shift + 1 : nk;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int64_t at = ((int64_t)m * a.H + h) * a.Nq + row[i];
      lse[m][i] = row[i] >= 0 ? a.lse[at] : kInf;
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
  f32x4 gq[2][QT][DQT];
#pragma unroll
  for (int i = 0; i < QT; ++i)
#pragma unroll
    for (int c = 0; c < DQT; ++c) gq[0][i][c] = gq[1][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int kb = 0; kb < last; kb += BK) {
    const int64_t base = (int64_t)k0 + kb;
    const uint8_t* keep = a.keep ? a.keep + base : nullptr;
    const int n = min(BK, nk - kb);
    auto ok = [&](int r) { return !keep || keep[r]; };
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m)
      stage<T, BK, DQ>(lk + m * DQ, LK, static_cast<const T*>(a.k) + base * a.k_rs + hk * a.k_hs + m * a.k_ms, a.k_rs, n, a.d, ok);
    stage<T, BK, DV>(lv, LV, static_cast<const T*>(a.v) + base * a.v_rs + hk * a.v_hs, a.v_rs, n, dv, ok);
    for (int r = threadIdx.x; r < BK; r += blockDim.x) lkeep[r] = r < n && ok(r);
    __syncthreads();

    f32x4 s[2][QT][2], dp[QT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < QT; ++i) s[0][i][u] = s[1][i][u] = dp[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const Frag<T> kf = frag_load(lk + (u * 16 + col) * LK + m * DQ + st * 32 + g * 8);
#pragma unroll
          for (int i = 0; i < QT; ++i) s[m][i][u] = mma(kf, qf[m][i][st], s[m][i][u]);
        }
#pragma unroll
      for (int st = 0; st < SV; ++st) {
        const Frag<T> vf = frag_load(lv + (u * 16 + col) * LV + st * 32 + g * 8);
#pragma unroll
        for (int i = 0; i < QT; ++i) dp[i][u] = mma(vf, of[i][st], dp[i][u]);
      }
      const int4 kp = *reinterpret_cast<const int4*>(lkeep + u * 16 + g * 4);
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = (&kp.x)[r] && kb + u * 16 + g * 4 + r < seen[i];
          const float p1 = in ? __builtin_amdgcn_exp2f(s[0][i][u][r] * scale2 - lse[0][i]) : 0.f;
          const float p2 = in ? lam * __builtin_amdgcn_exp2f(s[1][i][u][r] * scale2 - lse[1][i]) : 0.f;
          s[0][i][u][r] = p1 * (dp[i][u][r] - dl[0][i]);
          s[1][i][u][r] = -p2 * (dp[i][u][r] - dl[1][i]);
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      Frag<T> ds[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) ds[i] = frag_pack<T>(s[m][i][0], s[m][i][1]);
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const Frag<T> kf = frag_tr(lk, LK, 0, m * DQ + c * 16, lane);
#pragma unroll
        for (int i = 0; i < QT; ++i) gq[m][i][c] = mma(kf, ds[i], gq[m][i][c]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    if (row[i] < 0) continue;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < DQT; ++c) {
        const int x = c * 16 + g * 4;
        if (x < a.d) store4(static_cast<T*>(a.dq) + row[i] * a.dq_rs + h * a.dq_hs + m * a.dq_ms + x, gq[m][i][c] * a.scale);
      }
  }
}

// wavefronts of a workgroup whose wavefronts own `per_wave` rows, for segments of up to `longest` rows (0 = unknown)
int waves_for(int longest, int per_wave) { return longest <= 0 ? 4 : longest <= per_wave ? 1 : longest <= 2 * per_wave ? 2 : 4; }

template <typename T, int DQ, int RT>
void launch_bwd(const Args& a, hipStream_t s) {
  constexpr int per_wave = 16 * RT;
  const size_t tile = 32 * (4 * DQ + 2 * BCfg<T>::Pad) * sizeof(T);
  const int wk = waves_for(a.max_k, per_wave), wq = waves_for(a.max_q, per_wave);
  if (a.Nk > 0)
    k_diff_dkv<T, DQ, RT><<<dim3((unsigned)(a.Nk / (wk * per_wave) + a.B + 1), (unsigned)a.Hk), wk * 64, tile + 4 * 32 * sizeof(float), s>>>(a, a.ws);
  if (a.Nq > 0)
    k_diff_dq<T, DQ, RT><<<dim3((unsigned)(a.Nq / (wq * per_wave) + a.B + 1), (unsigned)a.H), wq * 64, tile + 32 * sizeof(int), s>>>(a, a.ws);
}

}  // namespace

// ws: delta [2, H, Nq] | partial sums of dlam [H, parts]
template <typename T>
void backward(const Args& a, hipStream_t s) {
  float* part = a.ws + (int64_t)2 * a.H * a.Nq;
  const int64_t parts = (a.Nq + kDeltaRows - 1) / kDeltaRows;
  if (a.Nq > 0) k_diff_delta<T><<<dim3((unsigned)parts, (unsigned)a.H), 256, 0, s>>>(a, a.ws, part);
  k_diff_dlam<T><<<(unsigned)a.H, 64, 0, s>>>(part, parts, a.dlam, a.lam_f32);
  if (a.d <= 32)
    launch_bwd<T, 32, 2>(a, s);
  else if (a.d <= 64)
    launch_bwd<T, 64, 2>(a, s);
  else
    launch_bwd<T, 128, 1>(a, s);
}

template void backward<float>(const Args&, hipStream_t);
template void backward<bf16>(const Args&, hipStream_t);
template void backward<f16>(const Args&, hipStream_t);

}  // namespace diffattn

extern "C" size_t gps_diff_attn_bwd_workspace_floats(int64_t Nq, int H) {
  if (Nq < 0 || H <= 0) return 0;
  return (size_t)H * (2 * (size_t)Nq + (size_t)((Nq + diffattn::kDeltaRows - 1) / diffattn::kDeltaRows));
}
