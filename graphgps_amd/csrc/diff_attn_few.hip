// Differential attention for few queries over long keys (diff_attn.hpp: formula, fragment layout, tile search): the keys are
// split, every part leaves its statistics and unnormalised sums, a second launch joins them.
//
// One WAVEFRONT per (unit of `cw` keys, key head): its 16 matrix columns are (query of the segment, head of the group) pairs, so
// the heads that share keys read them once.  K goes straight from memory into fragments; V passes through 32 rows of LDS that
// belong to the wavefront alone (no barrier anywhere) to be read down its columns.  Units are tiles of k_ptr: a long segment has more of
// them, none waits for another.  HBM-bound: K and V are read once.  One query over eight sequences of 33,000 keys, 8 heads over 2 of 64 columns, bf16:
// 268 MB in 57 us = 4.7 TB/s (a large copy: 4.88) and 9 us for the join; walking whole sequences in one workgroup took 17 ms.
#include "diff_attn.hpp"

namespace diffattn {
namespace {

constexpr int kUnitWaves = 4;

// statistics and sums of one unit, head and query: [2 dv] sums (map 1 | map 2), then m1, l1, m2, l2
__device__ __forceinline__ int64_t part_floats(int dv) { return 2 * dv + 4; }

template <typename T, int DQ>
__global__ __launch_bounds__(kUnitWaves * 64, sizeof(T) * DQ <= 128 ? 2 : 1) void k_diff_few(Args a, int cw, int cap) {
  constexpr int DV = 2 * DQ, DVT = DV / 16, ST = DQ / 32, LV = DV + 16 / (int)sizeof(T), El = 16 / sizeof(T);
  constexpr int NV = 32 * DV / El / 64;
  __shared__ __attribute__((aligned(16))) T lv_all[kUnitWaves][32 * LV];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
  T* lv = lv_all[wave];
  const int unit = blockIdx.x * kUnitWaves + wave, hk = blockIdx.y, group = a.H / a.Hk, dv = 2 * a.d;
  const Tile t = find_tile(a.k_ptr, a.B, a.Nk, cw, unit);
  if (t.rows <= 0 || t.seg >= a.B) return;
  const int q0 = clamp_row(a.q_ptr[t.seg], a.Nq), nq = max(0, clamp_row(a.q_ptr[t.seg + 1], a.Nq) - q0);
  const int shift = t.len - nq;
  const int cols = min(nq * group, cap);
  const float scale2 = a.scale * kLog2e;

  for (int c0 = 0; c0 < cols; c0 += 16) {
    const int c = c0 + col, qi = c / group, h = hk * group + c % group;
    const bool have = c < cols;
    const int seen = a.causal ? qi + shift + 1 - t.local : t.rows;   // keys of this unit that the column may see, by position
    Frag<T> q[2][ST];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        q[m][s] = frag_zero<T>();
        if (have && s * 32 + g * 8 < a.d)
          q[m][s] = frag_load(static_cast<const T*>(a.q) + (int64_t)(q0 + qi) * a.q_rs + h * a.q_hs + m * a.q_ms + s * 32 + g * 8);
      }
    f32x4 acc[2][DVT];
    float top[2] = {-kInf, -kInf}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < DVT; ++x) acc[0][x] = acc[1][x] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int kb = 0; kb < t.rows; kb += 32) {
      const int64_t base = (int64_t)t.first + kb;
      const int n = min(32, t.rows - kb);
      Frag<T> kf[2][2][ST];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = u * 16 + col;
        const bool ok = r < n && (!a.keep || a.keep[base + r]);
        const T* row = static_cast<const T*>(a.k) + (base + r) * a.k_rs + hk * a.k_hs + g * 8;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int s = 0; s < ST; ++s) {
            kf[m][u][s] = frag_zero<T>();
            if (ok && s * 32 + g * 8 < a.d) kf[m][u][s] = frag_load(row + m * a.k_ms + s * 32);
          }
      }
      uint4 vr[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = i * 64 + lane, r = at / (DV / El), x = at % (DV / El) * El;
        vr[i] = make_uint4(0, 0, 0, 0);
        if (r < n && x < dv && (!a.keep || a.keep[base + r]))
          vr[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + (base + r) * a.v_rs + hk * a.v_hs + x);
      }
      f32x4 s[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[m][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < ST; ++st) s[m][u] = mma(kf[m][u][st], q[m][st], s[m][u]);
        }
      // the wavefront's own LDS rows: its operations there are in order, the fences keep the compiler from moving them
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = i * 64 + lane;
        *reinterpret_cast<uint4*>(lv + at / (DV / El) * LV + at % (DV / El) * El) = vr[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      uint32_t dropped = 0;   // bit (u * 4 + r): key u * 16 + g * 4 + r is dropped
      if (a.keep) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = (j >> 2) * 16 + g * 4 + (j & 3);
          if (r < n && !a.keep[base + r]) dropped |= 1u << j;
        }
      }
      const int in = min(n, seen - kb);
      float f[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float hi = -kInf;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool see = u * 16 + g * 4 + r < in && !((dropped >> (u * 4 + r)) & 1u);
            s[m][u][r] = see ? s[m][u][r] * scale2 : -kInf;
            hi = maximum(hi, s[m][u][r]);
          }
        hi = over_groups(hi, [](float x, float y) { return maximum(x, y); });
        const float now = fmaxf(top[m], hi), off = now == -kInf ? 0.f : now;
        f[m] = __builtin_amdgcn_exp2f(top[m] - off);
        top[m] = now;
        float add = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[m][u][r] = __builtin_amdgcn_exp2f(s[m][u][r] - off);
            add += s[m][u][r];
          }
        sum[m] = sum[m] * f[m] + add;
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int x = 0; x < DVT; ++x) acc[m][x] *= f[m];
      }
      const Frag<T> p0 = frag_pack<T>(s[0][0], s[0][1]), p1 = frag_pack<T>(s[1][0], s[1][1]);
      Frag<T> lost0, lost1;   // weights in two terms, as in diff_attn.hip
      if constexpr (sizeof(T) == 2) {
        lost0 = frag_lost(s[0][0], s[0][1], p0);
        lost1 = frag_lost(s[1][0], s[1][1], p1);
      }
#pragma unroll
      for (int x = 0; x < DVT; ++x) {
        const Frag<T> vf = frag_tr(lv, LV, 0, x * 16, lane);
        acc[0][x] = mma(vf, p0, acc[0][x]);
        acc[1][x] = mma(vf, p1, acc[1][x]);
        if constexpr (sizeof(T) == 2) {
          acc[0][x] = mma(vf, lost0, acc[0][x]);
          acc[1][x] = mma(vf, lost1, acc[1][x]);
        }
      }
    }
    float* part = a.ws + (((int64_t)unit * a.Hk + hk) * cap + c) * part_floats(dv);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float z = over_groups(sum[m], [](float x, float y) { return x + y; });
      if (!have) continue;
#pragma unroll
      for (int x = 0; x < DVT; ++x)
        if (x * 16 + g * 4 < dv) *reinterpret_cast<f32x4*>(part + m * dv + x * 16 + g * 4) = acc[m][x];
      if (g == 0) {
        part[2 * dv + 2 * m] = top[m];
        part[2 * dv + 2 * m + 1] = z;
      }
    }
  }
}

// Joins the units of one (query row, head): weights 2^(m - M) of their sums, divided once.  A row past the `cap` columns that the
// units worked on (its segment has more queries than the caller said) is computed here from the definition.
template <typename T, int Waves>
__global__ __launch_bounds__(Waves * 64) void k_diff_join(Args a, int cw, int cap) {
  extern __shared__ float lds[];   // [Waves][2 dv], then [Waves][4]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, dv = 2 * a.d, group = a.H / a.Hk, hk = h / group;
  const int64_t row = blockIdx.x;
  float* stat = lds + Waves * 2 * dv;
  const int seg = find_segment(a.q_ptr, a.B, a.Nq, row);
  int q0 = 0, nq = 0, k0 = 0, nk = 0;
  if (seg < a.B) {
    q0 = clamp_row(a.q_ptr[seg], a.Nq);
    nq = max(0, clamp_row(a.q_ptr[seg + 1], a.Nq) - q0);
    k0 = clamp_row(a.k_ptr[seg], a.Nk);
    nk = max(0, clamp_row(a.k_ptr[seg + 1], a.Nk) - k0);
  }
  const int c = (int)(row - q0) * group + h % group;
  const bool direct = c >= cap;
  float m[2] = {-kInf, -kInf}, l[2] = {0.f, 0.f};
  float acc[2][4] = {};   // columns lane, lane + 64, ... of the two maps (dv <= 256)

  auto merge = [&](int i, float mu, float lu, float& keep, float& take) {   // running maximum over the units of this wavefront
    const float now = fmaxf(m[i], mu), ref = now == -kInf ? 0.f : now;
    keep = __builtin_amdgcn_exp2f(m[i] - ref);
    take = __builtin_amdgcn_exp2f(mu - ref);
    m[i] = now;
    l[i] = l[i] * keep + lu * take;
  };
  if (row >= q0 && row < (int64_t)q0 + nq && !direct) {
    const int first = k0 / cw + seg, count = (nk + cw - 1) / cw;
    for (int u = wave; u < count; u += Waves) {
      const float* part = a.ws + (((int64_t)(first + u) * a.Hk + hk) * cap + c) * part_floats(dv);
      const f32x4 ml = *reinterpret_cast<const f32x4*>(part + 2 * dv);
      float v[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) v[i][x] = x * 64 + lane < dv ? part[i * dv + x * 64 + lane] : 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float keep, take;
        merge(i, ml[2 * i], ml[2 * i + 1], keep, take);
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[i][x] = acc[i][x] * keep + v[i][x] * take;
      }
    }
  } else if (row >= q0 && row < (int64_t)q0 + nq) {
    const int see = a.causal ? min(nk, max(0, (int)(row - q0) + nk - nq + 1)) : nk;
    for (int j = wave; j < see; j += Waves) {
      const int64_t key = (int64_t)k0 + j;
      if (a.keep && !a.keep[key]) continue;
      for (int i = 0; i < 2; ++i) {
        float dot = 0.f;
        for (int x = lane; x < a.d; x += 64)
          dot += (float)static_cast<const T*>(a.q)[row * a.q_rs + h * a.q_hs + i * a.q_ms + x] *
                 (float)static_cast<const T*>(a.k)[key * a.k_rs + hk * a.k_hs + i * a.k_ms + x];
        for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
        float keep, take;
        merge(i, dot * a.scale * kLog2e, 1.f, keep, take);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          acc[i][x] = acc[i][x] * keep + (x * 64 + lane < dv ? take * (float)static_cast<const T*>(a.v)[key * a.v_rs + hk * a.v_hs + x * 64 + lane] : 0.f);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (x * 64 + lane < dv) lds[wave * 2 * dv + i * dv + x * 64 + lane] = acc[i][x];
    if (lane == 0) {
      stat[wave * 4 + 2 * i] = m[i];
      stat[wave * 4 + 2 * i + 1] = l[i];
    }
  }
  __syncthreads();
  const float lam = load_lam(a, h, static_cast<const T*>(nullptr));
  float w[2][Waves], lse[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float top = -kInf, z = 0.f;
#pragma unroll
    for (int j = 0; j < Waves; ++j) top = fmaxf(top, stat[j * 4 + 2 * i]);
    const float ref = top == -kInf ? 0.f : top;
#pragma unroll
    for (int j = 0; j < Waves; ++j) {
      w[i][j] = __builtin_amdgcn_exp2f(stat[j * 4 + 2 * i] - ref);
      z += w[i][j] * stat[j * 4 + 2 * i + 1];
    }
    const float inv = z == 0.f ? 0.f : 1.f / z;
    lse[i] = z == 0.f ? kInf : top + __builtin_amdgcn_logf(z);
#pragma unroll
    for (int j = 0; j < Waves; ++j) w[i][j] *= inv;
  }
  for (int x = threadIdx.x; x < dv; x += Waves * 64) {
    float o[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < Waves; ++j) o[i] += w[i][j] * lds[j * 2 * dv + i * dv + x];
    const int64_t at = (row * a.H + h) * dv + x;
    const float out = o[0] - lam * o[1];
    static_cast<T*>(a.o)[at] = (T)out;
    if constexpr (sizeof(T) == 2)
      if (a.o_rest) static_cast<T*>(a.o_rest)[at] = (T)(out - (float)(T)out);
    if (a.o2) a.o2[at] = o[1];
  }
  if (a.lse && threadIdx.x < 2) a.lse[((int64_t)threadIdx.x * a.H + h) * a.Nq + row] = threadIdx.x ? lse[1] : lse[0];
}

}  // namespace

// Keys per unit: about 1,024 units (4 wavefronts on each of 256 CUs) where the keys suffice.  One query over eight sequences of 33,000
// keys on average, 2 key heads of 64 columns, bf16, split + join: 512 units 92 + 7 us, 1,024 57 + 9, 2,048 62 + 14, 4,096 53 + 23.
int few_unit_keys(const Args& a) {
  int cw = 64;
  while (cw < 1024 && a.Nk * a.Hk > (int64_t)1024 * cw) cw *= 2;
  return cw;
}
int64_t few_units(const Args& a) { return a.Nk / few_unit_keys(a) + a.B + 1; }
int few_columns(const Args& a) { return a.max_q * (a.H / a.Hk); }

// Few queries: all (query, head of a group) pairs of a segment fit one column block, the keys do not fit one unit, and the join's grid
// of one workgroup per row stays far from the launch limit of 2^32 threads.  Two column blocks, each of which walks the unit's keys,
// where the form of diff_attn.hip would leave CUs idle, and in fp32, whose products are what takes the time.  Measured here / there (us;
// 64 columns, 4 heads of their own or 8 that share keys; forward):
//   columns  queries x keys x segments      bf16          fp32
//         1   1 x 65 x 2,000              75 / 100     225 / 527
//         1   1 x 400 x 300               48 / 52      247 / 280
//        32   4 x 4,000 x 8               26 / 144      42 / 488
//        32   32 x 4,000 x 8              57 / 144      93 / 488
//        32   4 x 1,000 x 64              71 / 64       95 / 259
//        32   32 x 4,000 x 64            257 / 197     873 / 974
bool few_applies(const Args& a) {
  const int columns = a.dtype == GPS_F32 || (int64_t)a.B * a.H < 256 ? 32 : 16;
  return a.max_q > 0 && a.max_q <= 32 && few_columns(a) <= columns && (a.max_k == 0 || a.max_k > 64) && a.Nk > 0 && a.Nq <= (1 << 20);
}
size_t few_workspace_floats(const Args& a) { return (size_t)few_units(a) * a.Hk * few_columns(a) * (4 * (size_t)a.d + 4); }

template <typename T>
void forward_few(const Args& a, hipStream_t s) {
  const int cw = few_unit_keys(a), cap = few_columns(a);
  const dim3 grid((unsigned)((few_units(a) + kUnitWaves - 1) / kUnitWaves), (unsigned)a.Hk);
  if (a.d <= 32)
    k_diff_few<T, 32><<<grid, kUnitWaves * 64, 0, s>>>(a, cw, cap);
  else if (a.d <= 64)
    k_diff_few<T, 64><<<grid, kUnitWaves * 64, 0, s>>>(a, cw, cap);
  else
    k_diff_few<T, 128><<<grid, kUnitWaves * 64, 0, s>>>(a, cw, cap);
  const size_t lds = (4 * a.d + 4) * sizeof(float);
  const dim3 rows((unsigned)a.Nq, (unsigned)a.H);
  // Long lists of units: 16 wavefronts walk one (33,000 keys on average, 2,048 units: 14 us against 35 with 4).  Short ones: 4 (32 queries
  // of ~125 keys: 4.1 us against 4.6).
  if (few_units(a) > (int64_t)16 * (a.B + 1))
    k_diff_join<T, 16><<<rows, 1024, 16 * lds, s>>>(a, cw, cap);
  else
    k_diff_join<T, 4><<<rows, 256, 4 * lds, s>>>(a, cw, cap);
}
template void forward_few<float>(const Args&, hipStream_t);
template void forward_few<bf16>(const Args&, hipStream_t);
template void forward_few<f16>(const Args&, hipStream_t);

}  // namespace diffattn
