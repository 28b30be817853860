// The residual stream of a block, in one pass over its rows:
//   n = norm(a; w1, b1)        y = alpha x + beta gate o n        z = norm(y; w2, b2)
// norm is LayerNorm or RMSNorm over the row; each of x, gate (a channel vector or a full matrix) and the two norms may be
// absent.  Backward, with r the reciprocal deviations, a^ and y^ the normalised rows and g' = g o w:
//   dyt = dy + r2 (dz' - y^ mean(dz' y^) - mean(dz')),  dx = alpha dyt,  dgate = beta dyt o n,
//   dn = beta dyt o gate,  da = r1 (dn' - a^ mean(dn' a^) - mean(dn'))       (the last mean only for LayerNorm)
//   dw2 = sum_rows dz o y^,  db2 = sum_rows dz,  dw1 = sum_rows dn o a^,  db1 = sum_rows dn.
//
// HBM-bound: forward 4 row streams (5 with a full gate), backward 6 (8).  A row lives in the registers of 16, 64 or 256 lanes,
// so that every element is read once; statistics are two-pass there (mean, then centred squares) in fp32, kept for the backward
// as four floats per row, and y is recomputed from x and a in fp32 rather than re-read rounded.  The column sums stay in
// registers while a workgroup walks its rows, leave once per workgroup, and a second launch adds them in a fixed order.
//
// 50,001 x 2,048, bf16, full gate: forward 191 us = 5.4 TB/s (a large copy: 4.88, half of it writes; here two streams in five),
// backward 386 us = 4.2 TB/s (the four sums' and the fetched row's registers leave two workgroups per CU), column sums 5 us.
// 7,681 x 384, fp32: 12.5, 23.5 and 4 us; a pass of both takes 160 us of host time.
#include "gps_common.hpp"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
using Args = gps_sandwich_norm;

constexpr int kThreads = 256;
constexpr int kSums = 5;          // dw1, db1, dw2, db2, dgate
constexpr int kCUs = 256;
constexpr int kGridX = 1 << 20;   // forward workgroups in one row of the grid (a grid dimension holds fewer than 2^32 threads)
constexpr int kMaxBlocks = 1024;  // most backward workgroups (= partial sums per column)

template <typename T, int V>
struct Chunk {
  typedef T Raw __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ Raw fetch(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void widen(const Raw& r, float* x) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (float)r[i];
  }
  static __device__ __forceinline__ void load(const T* p, float* x) {
    if constexpr (V == 1) {
      x[0] = (float)p[0];
    } else {
      typedef T vec __attribute__((ext_vector_type(V)));
      const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = (float)v[i];
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* x) {
    if constexpr (V == 1) {
      p[0] = (T)x[0];
    } else {
      typedef T vec __attribute__((ext_vector_type(V)));
      vec v;
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (T)x[i];
      *reinterpret_cast<vec*>(p) = v;
    }
  }
};

// parameters are fp32
template <int V>
__device__ __forceinline__ void load_param(const float* p, int c, float* x, float none) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = none;
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = p[c + i];
}

// sum over the TPR lanes of a row; every lane gets it.  sh: two floats per wavefront, `turn` alternates between two sets, so that
// one barrier per call is enough (a wavefront is at most one call ahead of the slowest reader).
template <int TPR>
__device__ __forceinline__ void row_sum2(float& x, float& y, float (*sh)[kThreads / 64][2], int& turn) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o; o >>= 1) {
    x += __shfl_xor(x, o);
    y += __shfl_xor(y, o);
  }
  if constexpr (TPR > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      sh[turn][w][0] = x;
      sh[turn][w][1] = y;
    }
    __syncthreads();
    x = y = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) {
      x += sh[turn][i][0];
      y += sh[turn][i][1];
    }
    turn ^= 1;
  }
}

// x -> (x - mean) * rstd over the row, in place; columns at and past D hold 0 on entry and keep no part in the sums
template <int TPR, int V, int NC>
__device__ __forceinline__ void normalise(float (&x)[NC][V], int lane, int D, bool layer, float eps, float& mean, float& rstd,
                                          float (*sh)[kThreads / 64][2], int& turn) {
  mean = 0.f;
  float none = 0.f;
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) s += x[c][i];
    row_sum2<TPR>(s, none, sh, turn);
    mean = s / (float)D;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const bool in = (c * TPR + lane) * V < D;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[c][i] = in ? x[c][i] - mean : 0.f;
      q += x[c][i] * x[c][i];
    }
  }
  none = 0.f;
  row_sum2<TPR>(q, none, sh, turn);
  rstd = 1.0f / sqrtf(q / (float)D + eps);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) x[c][i] *= rstd;
}

template <typename T, int TPR, int V, int NC>
__global__ __launch_bounds__(kThreads) void k_sandwich_fwd(Args a) {
  constexpr int RPB = kThreads / TPR;
  __shared__ float sh[2][kThreads / 64][2];
  int turn = 0;
  const int lane = threadIdx.x % TPR, D = a.D;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / TPR;
  if (row >= a.N) return;   // rows of one wavefront may leave here: sums are within the lanes of a row (TPR <= 64) or the
                            // whole workgroup has the same row (TPR = 256)
  const bool layer = a.kind == GPS_NORM_LAYER;
  float n[NC][V], w[V], b[V];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + lane) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) n[c][i] = 0.f;
    if (col < D) Chunk<T, V>::load(static_cast<const T*>(a.a) + row * a.a_rs + col, n[c]);
  }
  if (a.post_weight) {
    float mean, rstd;
    normalise<TPR, V, NC>(n, lane, D, layer, a.eps, mean, rstd, sh, turn);
    if (a.stats && lane == 0) {
      a.stats[row] = mean;
      a.stats[a.N + row] = rstd;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + lane) * V;
    if (col < D) {
      if (a.post_weight) {
        load_param<V>(a.post_weight, col, w, 1.f);
        load_param<V>(a.post_bias, col, b, 0.f);
#pragma unroll
        for (int i = 0; i < V; ++i) n[c][i] = n[c][i] * w[i] + b[i];
      }
      if (a.gate_full) {
        Chunk<T, V>::load(static_cast<const T*>(a.gate_full) + row * a.g_rs + col, w);
#pragma unroll
        for (int i = 0; i < V; ++i) n[c][i] *= w[i];
      } else if (a.gate) {
        load_param<V>(a.gate, col, w, 1.f);
#pragma unroll
        for (int i = 0; i < V; ++i) n[c][i] *= w[i];
      }
      if (a.x) {
        Chunk<T, V>::load(static_cast<const T*>(a.x) + row * a.x_rs + col, w);
#pragma unroll
        for (int i = 0; i < V; ++i) n[c][i] = a.alpha * w[i] + a.beta * n[c][i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) n[c][i] = a.beta * n[c][i];
      }
      Chunk<T, V>::store(static_cast<T*>(a.y) + row * D + col, n[c]);
    }
  }
  if (!a.pre_weight) return;
  float mean, rstd;
  normalise<TPR, V, NC>(n, lane, D, layer, a.eps, mean, rstd, sh, turn);
  if (a.stats && lane == 0) {
    a.stats[2 * a.N + row] = mean;
    a.stats[3 * a.N + row] = rstd;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + lane) * V;
    if (col < D) {
      load_param<V>(a.pre_weight, col, w, 1.f);
      load_param<V>(a.pre_bias, col, b, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) n[c][i] = n[c][i] * w[i] + b[i];
      Chunk<T, V>::store(static_cast<T*>(a.z) + row * D + col, n[c]);
    }
  }
}

template <typename T, int TPR, int V, int NC>
__global__ __launch_bounds__(kThreads) void k_sandwich_bwd(Args a) {
  constexpr int RPB = kThreads / TPR;
  __shared__ float sh[2][kThreads / 64][2];
  int turn = 0;
  const int lane = threadIdx.x % TPR, D = a.D;
  const bool layer = a.kind == GPS_NORM_LAYER, post = a.post_weight != nullptr, pre = a.pre_weight != nullptr;
  const float inv = 1.0f / (float)D;
  float acc[kSums][NC][V];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][c][i] = 0.f;

  // the next row's operands are fetched before this row's are used: between them lie two reductions over the row
  using C = Chunk<T, V>;
  struct Row {
    typename C::Raw a[NC], g[NC], x[NC], dz[NC], dy[NC];
    float m1, r1, m2, r2;
  };
  auto fetch = [&](int64_t row, Row& o) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * V;
      if (col >= D) continue;
      o.a[c] = C::fetch(static_cast<const T*>(a.a) + row * a.a_rs + col);
      if (a.gate_full) o.g[c] = C::fetch(static_cast<const T*>(a.gate_full) + row * a.g_rs + col);
      if (pre && a.x) o.x[c] = C::fetch(static_cast<const T*>(a.x) + row * a.x_rs + col);
      if (pre && a.dz) o.dz[c] = C::fetch(static_cast<const T*>(a.dz) + row * a.dz_rs + col);
      if (a.dy) o.dy[c] = C::fetch(static_cast<const T*>(a.dy) + row * a.dy_rs + col);
    }
    o.m1 = post ? a.stats[row] : 0.f;
    o.r1 = post ? a.stats[a.N + row] : 1.f;
    o.m2 = pre ? a.stats[2 * a.N + row] : 0.f;
    o.r2 = pre ? a.stats[3 * a.N + row] : 1.f;
  };
  const int64_t stride = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  Row next;
  if (row < a.N) fetch(row, next);
  for (; row < a.N; row += stride) {
    const Row R = next;
    if (row + stride < a.N) fetch(row + stride, next);
    const float m1 = R.m1, r1 = R.r1, m2 = R.m2, r2 = R.r2;
    float ah[NC][V], nn[NC][V], gt[NC][V], yh[NC][V], gz[NC][V], t[V], w[V], b[V];
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * V;
      const bool in = col < D;
#pragma unroll
      for (int i = 0; i < V; ++i) ah[c][i] = nn[c][i] = yh[c][i] = gz[c][i] = gt[c][i] = 0.f;
      if (!in) continue;
      C::widen(R.a[c], ah[c]);
#pragma unroll
      for (int i = 0; i < V; ++i) ah[c][i] = (ah[c][i] - m1) * r1;
      load_param<V>(a.post_weight, col, w, 1.f);
      load_param<V>(post ? a.post_bias : nullptr, col, b, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) nn[c][i] = post ? ah[c][i] * w[i] + b[i] : ah[c][i];
      if (a.gate_full)
        C::widen(R.g[c], gt[c]);
      else
        load_param<V>(a.gate, col, gt[c], 1.f);
      if (pre && a.dz) {
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = 0.f;
        if (a.x) C::widen(R.x[c], t);
        C::widen(R.dz[c], gz[c]);
        load_param<V>(a.pre_weight, col, w, 1.f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float y = a.alpha * t[i] + a.beta * (gt[c][i] * nn[c][i]);
          yh[c][i] = (y - m2) * r2;
          acc[2][c][i] += gz[c][i] * yh[c][i];
          acc[3][c][i] += gz[c][i];
          gz[c][i] *= w[i];
          s1 += gz[c][i] * yh[c][i];
          s0 += gz[c][i];
        }
      }
    }
    if (pre && a.dz) {
      row_sum2<TPR>(s0, s1, sh, turn);
      s0 = layer ? s0 * inv : 0.f;
      s1 *= inv;
    }
    float t0 = 0.f, t1 = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * V;
      if (col >= D) continue;
      float gy[V];
#pragma unroll
      for (int i = 0; i < V; ++i) gy[i] = 0.f;
      if (a.dy) C::widen(R.dy[c], gy);
      load_param<V>(a.post_weight, col, w, 1.f);
      float o1[V], o2[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        gy[i] += r2 * (gz[c][i] - yh[c][i] * s1 - s0);
        o1[i] = a.alpha * gy[i];
        const float gg = a.beta * gy[i];
        o2[i] = gg * nn[c][i];
        const float dn = gg * gt[c][i];
        acc[0][c][i] += dn * ah[c][i];
        acc[1][c][i] += dn;
        acc[4][c][i] += o2[i];
        gz[c][i] = post ? dn * w[i] : dn;   // from here on: dn'
        t1 += gz[c][i] * ah[c][i];
        t0 += gz[c][i];
      }
      if (a.dx) Chunk<T, V>::store(static_cast<T*>(a.dx) + row * D + col, o1);
      if (a.dgate_full) Chunk<T, V>::store(static_cast<T*>(a.dgate_full) + row * D + col, o2);
    }
    if (post) {
      row_sum2<TPR>(t0, t1, sh, turn);
      t0 = layer ? t0 * inv : 0.f;
      t1 *= inv;
    } else {
      t0 = t1 = 0.f;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * V;
      if (col >= D) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = r1 * (gz[c][i] - ah[c][i] * t1 - t0);
      Chunk<T, V>::store(static_cast<T*>(a.da) + row * D + col, o);
    }
  }

  // column sums of this workgroup -> ws[sum][workgroup][D]; the row slots of a workgroup meet in LDS, in slot order
  __shared__ float meet[kThreads * V];
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    float* out = a.ws + ((int64_t)k * gridDim.x + blockIdx.x) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + lane) * V;
      if constexpr (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) meet[threadIdx.x * V + i] = acc[k][c][i];
        __syncthreads();
        if (threadIdx.x < TPR) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float s = 0.f;
            for (int r = 0; r < RPB; ++r) s += meet[(r * TPR + lane) * V + i];
            acc[k][c][i] = s;
          }
        }
      }
      if (threadIdx.x < TPR && col < D) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[col + i] = acc[k][c][i];
      }
    }
  }
}

// column sums over the workgroups' partial sums: 64 columns x 16 slices of the partials per workgroup, eight loads in flight per
// thread (a slice of 64 dependent additions is latency, not bandwidth); slices meet in LDS, in order
__global__ __launch_bounds__(1024) void k_sandwich_cols(const float* __restrict__ ws, int parts, int D, float* o0, float* o1, float* o2,
                                                        float* o3, float* o4) {
  __shared__ float sh[16][64];
  float* outs[kSums] = {o0, o1, o2, o3, o4};
  float* out = outs[blockIdx.y];
  if (!out) return;
  const int x = threadIdx.x & 63, slice = threadIdx.x >> 6, c = blockIdx.x * 64 + x;
  const int per = (parts + 15) / 16, i0 = slice * per, i1 = min(parts, i0 + per);
  const float* p = ws + (int64_t)blockIdx.y * parts * D + min(c, D - 1);
  float s = 0.f;
  int i = i0;
  for (; i + 8 <= i1; i += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[(int64_t)(i + j) * D];
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[j];
  }
  for (; i < i1; ++i) s += p[(int64_t)i * D];
  sh[slice][x] = s;
  __syncthreads();
  if (slice == 0 && c < D) {
    s = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += sh[j][x];
    out[c] = s;
  }
}

int64_t rows_per_block(int tpr) { return kThreads / tpr; }
int blocks_for(int64_t N, int tpr) {
  const int64_t b = (N + rows_per_block(tpr) - 1) / rows_per_block(tpr);
  return (int)(b < kMaxBlocks ? b : kMaxBlocks);
}

template <typename T, int TPR, int V, int NC>
void launch(const Args& a, bool backward, hipStream_t s) {
  if (!backward) {
    const int64_t blocks = (a.N + rows_per_block(TPR) - 1) / rows_per_block(TPR);
    const unsigned x = (unsigned)(blocks < kGridX ? blocks : kGridX);
    k_sandwich_fwd<T, TPR, V, NC><<<dim3(x, (unsigned)((blocks + x - 1) / x)), kThreads, 0, s>>>(a);
    return;
  }
  // as many workgroups as are resident at once (a second, partly filled dispatch round would cost a whole row walk), each with an
  // equal share of the rows
  static const int resident = [] {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, reinterpret_cast<const void*>(&k_sandwich_bwd<T, TPR, V, NC>), kThreads, 0) != hipSuccess || n < 1) n = 1;
    return kCUs * n;
  }();
  const int most = blocks_for(a.N, TPR), blocks = most < resident ? most : resident;
  if (blocks > 0) k_sandwich_bwd<T, TPR, V, NC><<<blocks, kThreads, 0, s>>>(a);
  k_sandwich_cols<<<dim3((a.D + 63) / 64, kSums), 1024, 0, s>>>(a.ws, blocks, a.D, a.dpost_weight, a.dpost_bias, a.dpre_weight,
                                                               a.dpre_bias, a.dgate);
}

// Lanes of a row and chunks of V elements per lane, by the number of chunks.  Rows inside one wavefront need no barrier: 384 columns fp32 as
// 64 lanes x 2 chunks 12.4 us forward, 23.8 backward, as 256 lanes x 1 22.1 and 28.9; 64 columns as 16 lanes 4.3 us, as 64 lanes 4.6.
// Wider ones spread: 2,048 columns bf16 as 256 lanes x 1 chunk 191 and 386 us, as 64 x 4 191 and 500 (registers).
template <typename T, int V>
void by_width(const Args& a, bool backward, hipStream_t s) {
  const int chunks = (a.D + V - 1) / V;
  if (chunks <= 16) return launch<T, 16, V, 1>(a, backward, s);
  if (chunks <= 64) return launch<T, 64, V, 1>(a, backward, s);
  if (chunks <= 128) return launch<T, 64, V, 2>(a, backward, s);
  if constexpr (V <= 4)
    if (chunks <= 256) return launch<T, 64, V, 4>(a, backward, s);
  if (chunks <= 256) return launch<T, 256, V, 1>(a, backward, s);
  if (chunks <= 512) return launch<T, 256, V, 2>(a, backward, s);
  if (chunks <= 1024) return launch<T, 256, V, 4>(a, backward, s);
  if constexpr (V <= 4) {
    if (chunks <= 2048) return launch<T, 256, V, 8>(a, backward, s);
    if constexpr (V == 1) {   // widths that are no multiple of a 16-byte chunk, or unaligned rows
      if (chunks <= 4096) return launch<T, 256, V, 16>(a, backward, s);
      return launch<T, 256, V, 32>(a, backward, s);
    }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
void dispatch(const Args& a, bool backward, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.D % V == 0 && a.x_rs % V == 0 && a.a_rs % V == 0 && a.g_rs % V == 0 && a.dy_rs % V == 0 && a.dz_rs % V == 0 &&
                    aligned(a.x) && aligned(a.a) && aligned(a.gate_full) && aligned(a.y) && aligned(a.z) && aligned(a.dy) &&
                    aligned(a.dz) && aligned(a.dx) && aligned(a.da) && aligned(a.dgate_full);
  if (wide)
    by_width<T, V>(a, backward, s);
  else
    by_width<T, 1>(a, backward, s);
}

int check(const char* who, const Args* a) {
  GPS_REQUIRE(a != nullptr, "%s: null argument block", who);
  GPS_REQUIRE(a->dtype == GPS_F32 || a->dtype == GPS_BF16 || a->dtype == GPS_F16, "%s: dtype %d", who, a->dtype);
  GPS_REQUIRE(a->kind == GPS_NORM_RMS || a->kind == GPS_NORM_LAYER, "%s: kind %d", who, a->kind);
  GPS_REQUIRE(a->N >= 0 && a->N < (int64_t(1) << 31) && a->D > 0 && a->D <= gps_sandwich_max_width(), "%s: N=%lld D=%d", who, (long long)a->N, a->D);
  GPS_REQUIRE(!(a->gate && a->gate_full), "%s: two gates", who);
  GPS_REQUIRE(a->N == 0 || a->a, "%s: null pointer argument", who);
  return GPS_OK;
}

void dispatch_type(const Args& a, bool backward, hipStream_t s) {
  if (a.dtype == GPS_F32)
    dispatch<float>(a, backward, s);
  else if (a.dtype == GPS_BF16)
    dispatch<bf16>(a, backward, s);
  else
    dispatch<f16>(a, backward, s);
}

}  // namespace

extern "C" {

int gps_sandwich_max_width(void) { return 8192; }

size_t gps_sandwich_workspace_floats(int64_t N, int D) {
  if (N <= 0 || D <= 0) return 0;
  return (size_t)kSums * blocks_for(N, 256) * D;   // the row mapping with most workgroups
}

int gps_sandwich_norm_fwd(const gps_sandwich_norm* a, gps_stream_t stream) {
  if (const int rc = check("gps_sandwich_norm_fwd", a)) return rc;
  GPS_REQUIRE(a->N == 0 || (a->y && (!a->pre_weight || a->z)), "gps_sandwich_norm_fwd: null pointer argument");
  if (a->N == 0) return GPS_OK;
  dispatch_type(*a, false, gps::as_stream(stream));
  return gps::launch_status("gps_sandwich_norm_fwd");
}

int gps_sandwich_norm_bwd(const gps_sandwich_norm* a, gps_stream_t stream) {
  if (const int rc = check("gps_sandwich_norm_bwd", a)) return rc;
  GPS_REQUIRE(a->N == 0 || a->da, "gps_sandwich_norm_bwd: null pointer argument");
  GPS_REQUIRE(a->N == 0 || a->stats || !(a->post_weight || a->pre_weight), "gps_sandwich_norm_bwd: the forward's statistics are missing");
  const size_t need = gps_sandwich_workspace_floats(a->N, a->D);
  GPS_REQUIRE(need == 0 || (a->ws && a->ws_floats >= need), "gps_sandwich_norm_bwd: workspace of %zu floats, %zu needed", a->ws_floats, need);
  dispatch_type(*a, true, gps::as_stream(stream));
  return gps::launch_status("gps_sandwich_norm_bwd");
}

}  // extern "C"
