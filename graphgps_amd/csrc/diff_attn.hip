// Differential attention, forward (diff_attn.hpp: formula, fragment layout, tile search).
//
// One workgroup per (query tile, head): a wavefront owns QT x 16 queries, the workgroup walks the segment's keys in blocks of
// BN rows of K (both maps side by side) and V staged in LDS.  Scores are formed as S^T = K Q^T, so that a query is a lane's
// column: the running maximum and sum of each map need two cross-lane steps per block, the rescaling of the accumulators is by
// a per-lane scalar, and the weights feed O^T += V^T P^T from the registers they are in.  The two maps keep statistics and
// accumulators of their own and meet once, in the epilogue.
#include <initializer_list>

#include "diff_attn.hpp"

namespace {
using namespace diffattn;

template <typename T>
struct Cfg {
  static constexpr int BN = sizeof(T) == 4 ? 32 : 64;      // keys per block
  static constexpr int Pad = 16 / sizeof(T);               // row pitch of the LDS tiles: + 16 bytes
};

template <typename T, int DQ, int QT>
__global__ __launch_bounds__(256) void k_diff_fwd(Args a) {
  constexpr int DV = 2 * DQ, DVT = DV / 16, ST = DQ / 32, BN = Cfg<T>::BN, KT = BN / 16;
  constexpr int LK = 2 * DQ + Cfg<T>::Pad, LV = DV + Cfg<T>::Pad;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  T* lk = reinterpret_cast<T*>(lds_raw);
  T* lv = lk + BN * LK;
  int* lkeep = reinterpret_cast<int*>(lv + BN * LV);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
  const int bm = (blockDim.x >> 6) * 16 * QT, h = blockIdx.y, hk = h / (a.H / a.Hk), dv = 2 * a.d;
  const Tile t = find_tile(a.q_ptr, a.B, a.Nq, bm, blockIdx.x);
  if (t.rows <= 0) return;

  int k0 = 0, nk = 0;
  if (t.seg < a.B) {
    k0 = clamp_row(a.k_ptr[t.seg], a.Nk);
    nk = max(0, clamp_row(a.k_ptr[t.seg + 1], a.Nk) - k0);
  }
  const int shift = nk - t.len;   // causal: the query at index i of its segment sees keys <= i + shift
  const int last = a.causal ? min(nk, max(0, t.local + t.rows + shift)) : nk;

  Frag<T> q[2][QT][ST];
  int64_t row[QT];
  int seen[QT];                   // keys this lane's query may see, by position
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = (wave * QT + i) * 16 + col;
    const bool ok = r < t.rows;
    row[i] = ok ? t.first + r : -1;
    seen[i] = a.causal ? t.local + r + shift + 1 : nk;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        q[m][i][s] = frag_zero<T>();
        if (ok && s * 32 + g * 8 < a.d)
          q[m][i][s] = frag_load(static_cast<const T*>(a.q) + row[i] * a.q_rs + h * a.q_hs + m * a.q_ms + s * 32 + g * 8);
      }
  }
  f32x4 acc[2][QT][DVT];
  float top[2][QT], sum[2][QT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      top[m][i] = -kInf;
      sum[m][i] = 0.f;
#pragma unroll
      for (int c = 0; c < DVT; ++c) acc[m][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  const float scale2 = a.scale * kLog2e;

  for (int kb = 0; kb < last; kb += BN) {
    const int64_t base = (int64_t)k0 + kb;
    const uint8_t* keep = a.keep ? a.keep + base : nullptr;
    const int n = min(BN, nk - kb);
    auto ok = [&](int r) { return !keep || keep[r]; };
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m)
      stage<T, BN, DQ>(lk + m * DQ, LK, static_cast<const T*>(a.k) + base * a.k_rs + hk * a.k_hs + m * a.k_ms, a.k_rs, n, a.d, ok);
    stage<T, BN, DV>(lv, LV, static_cast<const T*>(a.v) + base * a.v_rs + hk * a.v_hs, a.v_rs, n, dv, ok);
    for (int r = threadIdx.x; r < BN; r += blockDim.x) lkeep[r] = r < n && ok(r);
    __syncthreads();

#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f32x4 s[QT][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int i = 0; i < QT; ++i) s[i][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const Frag<T> kf = frag_load(lk + (kt * 16 + col) * LK + m * DQ + st * 32 + g * 8);
#pragma unroll
          for (int i = 0; i < QT; ++i) s[i][kt] = mma(kf, q[m][i][st], s[i][kt]);
        }
      }
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        float hi = -kInf;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int4 kp = *reinterpret_cast<const int4*>(lkeep + kt * 16 + g * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool in = (&kp.x)[r] && kb + kt * 16 + g * 4 + r < seen[i];
            s[i][kt][r] = in ? s[i][kt][r] * scale2 : -kInf;
            hi = fmaxf(hi, s[i][kt][r]);
          }
        }
        hi = fmaxf(hi, __shfl_xor(hi, 16));
        hi = fmaxf(hi, __shfl_xor(hi, 32));
        const float now = fmaxf(top[m][i], hi);
        const float ref = now == -kInf ? 0.f : now;
        const float f = __builtin_amdgcn_exp2f(top[m][i] - ref);
        top[m][i] = now;
        float add = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[i][kt][r] = __builtin_amdgcn_exp2f(s[i][kt][r] - ref);
            add += s[i][kt][r];
          }
        sum[m][i] = sum[m][i] * f + add;
#pragma unroll
        for (int c = 0; c < DVT; ++c) acc[m][i][c] *= f;
      }
#pragma unroll
      for (int kk = 0; kk < BN / 32; ++kk) {
        Frag<T> p[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) p[i] = frag_pack<T>(s[i][2 * kk], s[i][2 * kk + 1]);
#pragma unroll
        for (int c = 0; c < DVT; ++c) {
          const Frag<T> vf = frag_tr(lv, LV, kk * 32, c * 16, lane);
#pragma unroll
          for (int i = 0; i < QT; ++i) acc[m][i][c] = mma(vf, p[i], acc[m][i][c]);
        }
      }
    }
  }

  const float lam = load_lam(a, h, static_cast<const T*>(nullptr));
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    float inv[2], l2[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float z = sum[m][i];
      z += __shfl_xor(z, 16);
      z += __shfl_xor(z, 32);
      inv[m] = z == 0.f ? 0.f : 1.f / z;
      l2[m] = z == 0.f ? kInf : top[m][i] + __builtin_amdgcn_logf(z);
    }
    if (row[i] < 0) continue;
    const int64_t at = (row[i] * a.H + h) * dv;
#pragma unroll
    for (int c = 0; c < DVT; ++c) {
      const int x = c * 16 + g * 4;
      if (x >= dv) continue;
      const f32x4 second = acc[1][i][c] * inv[1];
      store4(static_cast<T*>(a.o) + at + x, acc[0][i][c] * inv[0] - second * lam);
      if (a.o2) store4(a.o2 + at + x, second);
    }
    if (a.lse && g == 0) {
      a.lse[(int64_t)h * a.Nq + row[i]] = l2[0];
      a.lse[((int64_t)a.H + h) * a.Nq + row[i]] = l2[1];
    }
  }
}

template <typename T, int DQ, int QT>
void launch_fwd(const Args& a, hipStream_t s) {
  const int per_wave = 16 * QT;
  const int waves = a.max_q > 0 && a.max_q <= per_wave ? 1 : a.max_q > 0 && a.max_q <= 2 * per_wave ? 2 : 4;
  const dim3 grid((unsigned)(a.Nq / (waves * per_wave) + a.B + 1), (unsigned)a.H);
  const size_t lds = Cfg<T>::BN * ((4 * DQ + 2 * Cfg<T>::Pad) * sizeof(T) + sizeof(int));
  k_diff_fwd<T, DQ, QT><<<grid, waves * 64, lds, s>>>(a);
}

template <typename T>
void forward(const Args& a, hipStream_t s) {
  if (few_applies(a))
    forward_few<T>(a, s);
  else if (a.d <= 32)
    launch_fwd<T, 32, 2>(a, s);
  else if (a.d <= 64)
    launch_fwd<T, 64, 2>(a, s);
  else
    launch_fwd<T, 128, 1>(a, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool by8(std::initializer_list<int64_t> strides) {
  for (int64_t x : strides)
    if (x % 8 != 0) return false;
  return true;
}

// what both entry points ask of their arguments
int check(const char* who, const Args* a) {
  GPS_REQUIRE(a != nullptr, "%s: null argument block", who);
  GPS_REQUIRE(a->dtype == GPS_F32 || a->dtype == GPS_BF16 || a->dtype == GPS_F16, "%s: dtype %d", who, a->dtype);
  GPS_REQUIRE(a->B >= 0 && a->H > 0 && a->Hk > 0 && a->H % a->Hk == 0 && a->H <= 65535, "%s: B=%d H=%d Hk=%d", who, a->B, a->H, a->Hk);
  GPS_REQUIRE(a->d > 0 && a->d <= 128 && a->d % 8 == 0, "%s: d=%d is no multiple of 8 up to 128", who, a->d);
  GPS_REQUIRE(a->Nq >= 0 && a->Nk >= 0 && a->Nq < (int64_t(1) << 31) && a->Nk < (int64_t(1) << 31), "%s: Nq=%lld Nk=%lld", who,
              (long long)a->Nq, (long long)a->Nk);
  GPS_REQUIRE(a->max_q >= 0 && a->max_k >= 0, "%s: max_q=%d max_k=%d", who, a->max_q, a->max_k);
  GPS_REQUIRE(a->q_ptr && a->k_ptr && a->lam, "%s: null pointer argument", who);
  GPS_REQUIRE(a->Nq == 0 || (a->q && a->o), "%s: null pointer argument", who);
  GPS_REQUIRE(a->Nk == 0 || (a->k && a->v), "%s: null pointer argument", who);
  GPS_REQUIRE(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->o) && aligned16(a->o2) && aligned16(a->ws), "%s: pointers must be 16-byte aligned", who);
  GPS_REQUIRE(by8({a->q_rs, a->q_hs, a->q_ms, a->k_rs, a->k_hs, a->k_ms, a->v_rs, a->v_hs}), "%s: strides must be multiples of 8 elements", who);
  GPS_REQUIRE((a->o2 == nullptr) == (a->lse == nullptr), "%s: o2 and lse come together", who);
  return GPS_OK;
}

}  // namespace

extern "C" {

size_t gps_diff_attn_fwd_workspace_floats(const gps_diff_attn* a) {
  if (!a || a->H <= 0 || a->Hk <= 0 || a->Nq <= 0 || !few_applies(*a)) return 0;
  return few_workspace_floats(*a);
}

int gps_diff_attn_fwd(const gps_diff_attn* a, gps_stream_t stream) {
  if (const int rc = check("gps_diff_attn_fwd", a)) return rc;
  if (a->Nq == 0) return GPS_OK;
  const size_t need = gps_diff_attn_fwd_workspace_floats(a);
  GPS_REQUIRE(need == 0 || (a->ws && a->ws_floats >= need), "gps_diff_attn_fwd: workspace of %zu floats, %zu needed", a->ws_floats, need);
  hipStream_t s = gps::as_stream(stream);
  if (a->dtype == GPS_F32)
    forward<float>(*a, s);
  else if (a->dtype == GPS_BF16)
    forward<bf16>(*a, s);
  else
    forward<f16>(*a, s);
  return gps::launch_status("gps_diff_attn_fwd");
}

int gps_diff_attn_bwd(const gps_diff_attn* a, gps_stream_t stream) {
  if (const int rc = check("gps_diff_attn_bwd", a)) return rc;
  GPS_REQUIRE(a->dlam, "gps_diff_attn_bwd: null pointer argument");
  GPS_REQUIRE(a->Nq == 0 || (a->o2 && a->dout && a->dq), "gps_diff_attn_bwd: null pointer argument");
  GPS_REQUIRE(a->Nk == 0 || (a->dk && a->dv), "gps_diff_attn_bwd: null pointer argument");
  GPS_REQUIRE(aligned16(a->dout) && aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv) &&
                  by8({a->do_rs, a->do_hs, a->dq_rs, a->dq_hs, a->dq_ms, a->dk_rs, a->dk_hs, a->dk_ms, a->dv_rs, a->dv_hs}),
              "gps_diff_attn_bwd: gradients must be 16-byte aligned, their strides multiples of 8 elements");
  const size_t need = gps_diff_attn_bwd_workspace_floats(a->Nq, a->H);
  GPS_REQUIRE(need == 0 || (a->ws && a->ws_floats >= need), "gps_diff_attn_bwd: workspace of %zu floats, %zu needed", a->ws_floats, need);
  hipStream_t s = gps::as_stream(stream);
  if (a->dtype == GPS_F32)
    backward<float>(*a, s);
  else if (a->dtype == GPS_BF16)
    backward<bf16>(*a, s);
  else
    backward<f16>(*a, s);
  return gps::launch_status("gps_diff_attn_bwd");
}

}  // extern "C"
