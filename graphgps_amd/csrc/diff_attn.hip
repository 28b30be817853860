// Differential attention, forward (diff_attn.hpp: formula, fragment layout, tile search).
//
// One workgroup per (query tile, head): a wavefront owns QT x 16 queries, the workgroup walks the segment's keys in blocks of
// BN rows of K (both maps side by side) and V staged in LDS.  Scores are formed as S^T = K Q^T, so that a query is a lane's
// column: the running maximum and sum of each map need two cross-lane steps per block, the rescaling of the accumulators is by
// a per-lane scalar, and the weights feed O^T += V^T P^T from the registers they are in.  The two maps keep statistics and
// accumulators of their own and meet once, in the epilogue.  Two blocks of K and V are in LDS: one is read while the next one arrives,
// straight from memory, behind a single barrier per block.
//
// In 16 bits a weight enters the second product in two terms, its rounding and what that lost (frag_lost).  The maps nearly cancel where
// they agree, and a single rounding of each leaves its error on that small difference: relative to the value rounded once at the end, the
// error of o is 1.0 times with two terms and 1.4 to 1.55 times with one on independent maps (0.0017 against 0.0025; two graphs of ~4,700
// nodes 478 against 353 us, trees 14.1 against 11.7, ordered sequences 403 against 373), and 1 / (1 - lam) times and more where they
// resemble each other.  Rounding the difference of the maps' weights instead needs the ratio of their final sums while it is formed: a
// ratio from the keys seen so far puts errors into the sum that go by a key's weight when it was met, not by its weight at the end.
//
// Bound by the matrix units and what a SIMD issues around them: at 64 columns a block of 16 x 32 pairs is 40 matrix instructions (16
// cycles each) and about 180 vector instructions, two exponentials per pair among them.  Two graphs of 4,175 and 5,261 nodes, 8 heads over
// 4 of 64 columns, bf16: 478 us = 970 TFLOP/s of the products that the kernel makes (20 d flops per pair and head; 8 d are the
// operator's), where a large matrix product reaches 1,262.  Four causal sequences of ~2,600 rows, 6 heads over 2 of 128 columns, fp16,
// dropped keys: 403 us.  256 molecules of ~31 nodes, 8 heads of 24 columns, fp32: 42 us; 32 trees of ~123 nodes, 4 heads of 32, bf16: 14.1.
#include <initializer_list>

#include "diff_attn.hpp"

namespace {
using namespace diffattn;

// Keys per block: 64 where the registers hold three wavefronts per SIMD with it, else 32.  16 bits, 32 columns (syntax trees of ~125 nodes):
// 14.5 us with 64, 14.9 with 32, and 16.9 against 19.6 with dropped keys; 64 columns (two graphs of ~4,700 nodes): 775 with 64, 497 with
// 32; fp32, 32 columns (molecules): 66 with 64, 42 with 32.
template <typename T, int DQ>
constexpr int block_keys() { return sizeof(T) * DQ <= 64 ? 64 : 32; }

// A row's largest weight is 2^kUp when its reference is set.  float16 weights below 2^-25 round to zero, and a long row may have a share
// of its sum in keys that far below its largest, so the largest is put near the top of the type (2^(9 + 6) < 65504).
template <typename T>
constexpr float kUp = 0.f;
template <>
constexpr float kUp<f16> = 9.f;

template <typename T, int DQ, int QT, bool Masked>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (QT == 1 && DQ <= 64 ? 3 : 2) : DQ == 32 ? 3 : 1) void k_diff_fwd(Args a, int tile_count) {
  constexpr int DV = 2 * DQ, DVT = DV / 16, ST = DQ / 32, BN = block_keys<T, DQ>(), KT = BN / 16;
  typedef Tl<T, DV> L;   // rows of K (both maps) and of V have the same width
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds_raw[];
  T* tiles = reinterpret_cast<T*>(lds_raw);                  // [2][K | V]
  int* lkeep = reinterpret_cast<int*>(tiles + 4 * BN * DV);  // [2][BN]

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
  const Unit unit = xcd_unit(blockIdx.x, tile_count, a.H);
  if (unit.tile >= tile_count || unit.head >= a.H) return;
  const int bm = (blockDim.x >> 6) * 16 * QT, h = unit.head, hk = h / (a.H / a.Hk), dv = 2 * a.d;
  const Tile t = find_tile(a.q_ptr, a.B, a.Nq, bm, unit.tile);
  if (t.rows <= 0) return;

  int k0 = 0, nk = 0;
  if (t.seg < a.B) {
    k0 = clamp_row(a.k_ptr[t.seg], a.Nk);
    nk = max(0, clamp_row(a.k_ptr[t.seg + 1], a.Nk) - k0);
  }
  const int shift = nk - t.len;   // causal: the query at index i of its segment sees keys <= i + shift
  const int last = a.causal ? min(nk, max(0, t.local + t.rows + shift)) : nk;

  const RowShare<BN> share;
  bool kept = true;   // whether this thread's row of the block that was fetched last is a key
  const Stager<T, BN, DV, 2> stage_k(a.k_rs, a.k_ms, a.d);
  const Stager<T, BN, DV, 1> stage_v(a.v_rs, 0, dv);
  auto fetch = [&](int kb, int buf) __attribute__((always_inline)) {
    T* lk = tiles + buf * 2 * BN * DV;
    const int64_t base = (int64_t)k0 + kb;
    const int n = min(BN, nk - kb);
    const T* ks = static_cast<const T*>(a.k) + base * a.k_rs + hk * a.k_hs;
    const T* vs = static_cast<const T*>(a.v) + base * a.v_rs + hk * a.v_hs;
    if constexpr (Masked) kept = share.row < n && a.keep[base + min(share.row, n - 1)];
    stage_k(lk, ks, a.k_rs, a.k_ms, n, a.d);
    stage_v(lk + BN * DV, vs, a.v_rs, 0, n, dv);
  };
  if (last > 0) fetch(0, 0);

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
  const int all_see = a.causal ? t.local + wave * QT * 16 + shift + 1 : nk;   // keys that every query of this wavefront sees
  f32x4 acc[2][QT][DVT];   // of each map: sum p v with p = 2^(score - ref)
  float ref[2][QT], sum[2][QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      ref[m][i] = -kLowest;
      sum[m][i] = 0.f;
#pragma unroll
      for (int c = 0; c < DVT; ++c) acc[m][i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  const float scale2 = a.scale * kLog2e, lam = load_lam(a, h, static_cast<const T*>(nullptr));

  int buf = 0;
  for (int kb = 0; kb < last; kb += BN, buf ^= 1) {
    tiles_ready();
    const T* lk = tiles + buf * 2 * BN * DV;
    const T* lv = lk + BN * DV;
    if constexpr (Masked) {   // scores of dropped keys are cut below; their rows of V would meet weights of 0
      if (!kept) share.template zero<T, DV>(const_cast<T*>(lv));
      if (share.part == 0) lkeep[buf * BN + share.row] = kept;
      __syncthreads();
    }
    if (kb + BN < last) fetch(kb + BN, buf ^ 1);
    f32x4 s[2][QT][KT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int i = 0; i < QT; ++i) s[m][i][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const Frag<T> kf = L::frag(lk, kt * 16 + col, m * DQ + st * 32 + g * 8);
#pragma unroll
          for (int i = 0; i < QT; ++i) s[m][i][kt] = mma(kf, q[m][i][st], s[m][i][kt]);
        }
      }
    if (Masked || kb + BN > all_see) {   // (uniform over the wavefront)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        int4 kp = make_int4(1, 1, 1, 1);
        if constexpr (Masked) kp = *reinterpret_cast<const int4*>(lkeep + buf * BN + kt * 16 + g * 4);
#pragma unroll
        for (int i = 0; i < QT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool in = (&kp.x)[r] && kb + kt * 16 + g * 4 + r < seen[i];
            s[0][i][kt][r] = in ? s[0][i][kt][r] : -kInf;
            s[1][i][kt][r] = in ? s[1][i][kt][r] : -kInf;
          }
      }
    }
    // The references move only when a score passes one by more than 6 + kUp: weights stay below 2^(6 + kUp), inside every type, and
    // the accumulators are rescaled a few times per row instead of at every new maximum.
    float hi[2][QT];   // over this lane's keys
    bool past = false;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        float x = s[m][i][0][0];
#pragma unroll
        for (int j = 1; j + 1 < 4 * KT; j += 2) x = maximum(maximum(x, s[m][i][j / 4][j % 4]), s[m][i][(j + 1) / 4][(j + 1) % 4]);
        hi[m][i] = maximum(x, s[m][i][KT - 1][3]);
        past |= __builtin_fmaf(hi[m][i], scale2, -ref[m][i]) > 6.f + kUp<T>;
      }
    const bool move = __any(past);
    float f[2][QT];
    if (move) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          const float now = fmaxf(ref[m][i], over_groups(hi[m][i], [](float u, float v) { return maximum(u, v); }) * scale2 - kUp<T>);
          f[m][i] = __builtin_amdgcn_exp2f(ref[m][i] - now);
          ref[m][i] = now;
          sum[m][i] *= f[m][i];
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        float add = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[m][i][kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][i][kt][r], scale2, -ref[m][i]));
            add += s[m][i][kt][r];
          }
        sum[m][i] += add;
      }
    Frag<T> p[2][QT][BN / 32], lost[2][QT][BN / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        if (move) {
#pragma unroll
          for (int c = 0; c < DVT; ++c) acc[m][i][c] *= f[m][i];
        }
#pragma unroll
        for (int kk = 0; kk < BN / 32; ++kk) {
          p[m][i][kk] = frag_pack<T>(s[m][i][2 * kk], s[m][i][2 * kk + 1]);
          if constexpr (sizeof(T) == 2) lost[m][i][kk] = frag_lost(s[m][i][2 * kk], s[m][i][2 * kk + 1], p[m][i][kk]);
        }
      }
#pragma unroll
    for (int kk = 0; kk < BN / 32; ++kk)
#pragma unroll
      for (int c = 0; c < DVT; ++c) {
        const Frag<T> vf = L::frag_tr(lv, kk * 32, c * 16, lane);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          acc[0][i][c] = mma(vf, p[0][i][kk], acc[0][i][c]);
          acc[1][i][c] = mma(vf, p[1][i][kk], acc[1][i][c]);
          if constexpr (sizeof(T) == 2) {
            acc[0][i][c] = mma(vf, lost[0][i][kk], acc[0][i][c]);
            acc[1][i][c] = mma(vf, lost[1][i][kk], acc[1][i][c]);
          }
        }
      }
  }

#pragma unroll
  for (int i = 0; i < QT; ++i) {
    float inv[2], l2[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float z = over_groups(sum[m][i], [](float u, float v) { return u + v; });
      inv[m] = z == 0.f ? 0.f : 1.f / z;
      l2[m] = z == 0.f ? kInf : ref[m][i] + __builtin_amdgcn_logf(z);
    }
    if (row[i] < 0) continue;
    const int64_t at = (row[i] * a.H + h) * dv;
#pragma unroll
    for (int c = 0; c < DVT; ++c) {
      const int x = c * 16 + g * 4;
      if (x >= dv) continue;
      store_out4<T>(a, at + x, acc[0][i][c] * inv[0] - acc[1][i][c] * (lam * inv[1]));
      if (a.o2) store4(a.o2 + at + x, acc[1][i][c] * inv[1]);
    }
    if (a.lse && g == 0) {
      a.lse[(int64_t)h * a.Nq + row[i]] = l2[0];
      a.lse[((int64_t)a.H + h) * a.Nq + row[i]] = l2[1];
    }
  }
}

// QT = 1 everywhere: two tiles per wavefront halve its LDS reads but take the third wavefront's registers (two graphs of ~4,700
// nodes, 64 columns: 786 us against 497; trees 17.0 against 14.5; molecules in fp32: 62 against 42).
template <typename T, int DQ, int QT>
void launch_fwd(const Args& a, hipStream_t s) {
  const int per_wave = 16 * QT;
  // Short segments: a workgroup as tall as the longest, no idle wavefronts in its barriers.  fp32, 8 heads of 24 columns: 1,024 graphs of 15
  // nodes 73 us with 1, 79 with 2, 90 with 4; 512 of 30 nodes 49 with 2, 53 with 4 (the backward: 179, 185, 237 and 118, 140).
  const int waves = a.max_q > 0 && a.max_q <= per_wave ? 1 : a.max_q > 0 && a.max_q <= 2 * per_wave ? 2 : 4;
  const int tiles = (int)(a.Nq / (waves * per_wave)) + a.B + 1;
  const unsigned grid = (unsigned)xcd_grid(tiles * a.H);
  const size_t lds = 2 * block_keys<T, DQ>() * (4 * DQ * sizeof(T) + (a.keep ? sizeof(int) : 0));
  if (a.keep)
    k_diff_fwd<T, DQ, QT, true><<<grid, waves * 64, lds, s>>>(a, tiles);
  else
    k_diff_fwd<T, DQ, QT, false><<<grid, waves * 64, lds, s>>>(a, tiles);
}

template <typename T>
void forward(const Args& a, hipStream_t s) {
  if (few_applies(a))
    forward_few<T>(a, s);
  else if (a.d <= 32)
    launch_fwd<T, 32, 1>(a, s);
  else if (a.d <= 64)
    launch_fwd<T, 64, 1>(a, s);
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
  // the launch grids: tiles of 16 rows at least, 256 threads at most, below 2^32 threads
  GPS_REQUIRE((a->Nq / 16 + a->B + 1) * a->H + (a->Nk / 16 + a->B + 1) * a->Hk + a->H < (int64_t(1) << 24), "%s: Nq=%lld Nk=%lld B=%d: more tiles than one launch holds",
              who, (long long)a->Nq, (long long)a->Nk, a->B);
  GPS_REQUIRE(a->scale > 0.f && a->scale < kInf, "%s: scale %g is not positive", who, (double)a->scale);
  GPS_REQUIRE(a->max_q >= 0 && a->max_k >= 0, "%s: max_q=%d max_k=%d", who, a->max_q, a->max_k);
  GPS_REQUIRE(a->q_ptr && a->k_ptr && a->lam, "%s: null pointer argument", who);
  GPS_REQUIRE(a->Nq == 0 || (a->q && a->o), "%s: null pointer argument", who);
  GPS_REQUIRE(a->Nk == 0 || (a->k && a->v), "%s: null pointer argument", who);
  GPS_REQUIRE(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->o) && aligned16(a->o2) && aligned16(a->o_rest) && aligned16(a->ws), "%s: pointers must be 16-byte aligned", who);
  GPS_REQUIRE(by8({a->q_rs, a->q_hs, a->q_ms, a->k_rs, a->k_hs, a->k_ms, a->v_rs, a->v_hs}), "%s: strides must be multiples of 8 elements", who);
  // the lanes' offsets within a block of rows are 32-bit
  for (int64_t x : {a->q_rs, a->k_rs, a->v_rs, a->do_rs}) GPS_REQUIRE(x >= 0 && x <= (1 << 22), "%s: row stride %lld", who, (long long)x);
  for (int64_t x : {a->q_ms, a->k_ms}) GPS_REQUIRE(x >= 0 && x <= (1 << 28), "%s: map stride %lld", who, (long long)x);
  GPS_REQUIRE((a->o2 == nullptr) == (a->lse == nullptr), "%s: o2 and lse come together", who);
  GPS_REQUIRE(!a->o_rest || a->dtype != GPS_F32, "%s: o_rest is for 16-bit types", who);
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
  const size_t need = gps_diff_attn_bwd_workspace_floats(a->Nq, a->H, a->B);
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
