// Gradient-norm clip + AdamW over the flat parameter arena with both moments in 8 bits (format: include/gps_hip.h).
//
// HBM-bound: p read and written, g read (twice with the norm), a byte read and written for each moment = 20 B per parameter
// against 32 with fp32 moments.  A wavefront owns one quantisation block of 256 elements, four per lane: its new maximum is one
// cross-lane reduction, nothing is written before it is known, and no block is visited twice.
//   K1 k_sqnorm8 : per-workgroup sums of g^2 over a bounded number of workgroups (so that K2 can re-add them all); works out each
//                  chunk's bias corrections (two fp64 powers: in K2 they would cost every workgroup their registers)
//                  200 M parameters: 800 MB in 180 us = 4.4 TB/s (a chunk's four loads per thread are issued together: 205 one by one)
//   K2 k_adamw8  : every workgroup adds K1's sums in the same order (fp64) -> clip coefficient, then updates its chunks; a
//                  parameter's first chunk advances its step counter.  200 M: 3.2 GB in 780-810 us = 4.0 TB/s (a large copy:
//                  4.88), 19 M: 73 us.  Tried without gain: the next block fetched ahead (787), five wavefronts per SIMD instead of four (797, spilling)
// k_adamw8_values: both moments of 200 M parameters as bf16, 1.2 GB in 196 us = 6.1 TB/s
#include "gps_common.hpp"

namespace {

constexpr int kChunk = 4096;   // = gps_optim_chunk()
constexpr int kBlock = 256;    // elements that share a unit
constexpr int kPer = kChunk / kBlock;
constexpr int kThreads = 256, kWaves = kThreads / 64;
// 200 M parameters: norm 180 us with 1,024 workgroups, 197 with 2,048; step within 2 % from 2,048 to 8,192 (1,024: 1 % slower)
constexpr int kNormBlocks = 1024, kStepBlocks = 2048;

enum { H_LR = 0, H_B1, H_B2, H_EPS, H_WD, H_MAXNORM, H_STEP, H_NORM, H_COUNT };

struct ChunkCoef {   // one chunk's step number (its parameter's) and bias corrections
  float step, size, inv_bc2_sqrt;
};

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16; x *= 0x7feb352dU; x ^= x >> 15; x *= 0x846ca68bU; x ^= x >> 16;
  return x;
}

__global__ __launch_bounds__(kThreads) void k_sqnorm8(const float* __restrict__ g, const int64_t* __restrict__ chunk_off,
                                                      const int32_t* __restrict__ chunk_len, const int32_t* __restrict__ chunk_param,
                                                      const uint8_t* __restrict__ active, int64_t n_chunks,
                                                      double* __restrict__ hyper, const float* __restrict__ pstep,
                                                      float* __restrict__ ws, ChunkCoef* __restrict__ coef) {
  __shared__ float sh[kWaves];
  int known = -1;   // the parameter that `mine` is of (thread 0)
  ChunkCoef mine = {};
  if (blockIdx.x == 0 && threadIdx.x == 0) hyper[H_STEP] += 1.0;
  float acc = 0.f;
  for (int64_t c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const int prm = chunk_param[c];
    if (!active[prm]) continue;
    if (threadIdx.x == 0) {
      if (prm != known) {
        known = prm;
        mine.step = pstep[prm] + 1.0f;
        mine.size = (float)(hyper[H_LR] / (1.0 - pow(hyper[H_B1], (double)mine.step)));
        mine.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - pow(hyper[H_B2], (double)mine.step)));
      }
      coef[c] = mine;
    }
    const float* gp = g + chunk_off[c];
    const int len = chunk_len[c];
    const int n4 = (reinterpret_cast<uintptr_t>(gp) & 15) == 0 ? len >> 2 : 0;
    if (n4 == kChunk / 4) {   // the usual chunk
      float4 x[kChunk / 4 / kThreads];
#pragma unroll
      for (int j = 0; j < kChunk / 4 / kThreads; ++j) x[j] = reinterpret_cast<const float4*>(gp)[j * kThreads + threadIdx.x];
#pragma unroll
      for (int j = 0; j < kChunk / 4 / kThreads; ++j) acc += x[j].x * x[j].x + x[j].y * x[j].y + x[j].z * x[j].z + x[j].w * x[j].w;
    } else {
      for (int i = threadIdx.x; i < n4; i += kThreads) {
        const float4 x = reinterpret_cast<const float4*>(gp)[i];
        acc += x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
      }
    }
    for (int i = (n4 << 2) + threadIdx.x; i < len; i += kThreads) acc += gp[i] * gp[i];
  }
  for (int o = 32; o; o >>= 1) acc += __shfl_xor(acc, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) ws[blockIdx.x] = sh[0] + sh[1] + sh[2] + sh[3];
}

// value of a magnitude code, in units
__device__ __forceinline__ float units_of(uint32_t c) { return c < 8u ? (float)c : __uint_as_float((c + 1032u) << 20); }
__device__ __forceinline__ float unit_of(uint32_t e) { return __uint_as_float(e << 23); }

// exponent byte of a block from the bits of its largest magnitude; `octaves`: the unit keeps values up to 15 * 2^(octaves - 4)
__device__ __forceinline__ int unit_exponent(uint32_t top, int octaves) {
  if (top == 0u) return 0;
  if (top >= 0x7f800000u) return 255;
  const int k = (int)(top >> 23) - 126 + ((top & 0x7fffffu) > 0x700000u ? 1 : 0) - octaves;
  return (k < -126 ? -126 : k) + 127;
}
// magnitude of y units -> code, rounded up with probability r / 65536 of the way to the next one
__device__ __forceinline__ uint32_t code_of(float y, uint32_t r) {
  return y < 8.f ? (uint32_t)floorf(y + (float)r * 0x1p-16f) : ((__float_as_uint(y) + (r << 4)) >> 20) - 1032u;
}

struct Coef {
  float decay, one_m_b1, b2, one_m_b2, eps, clip;
};

// One element; m and v leave unrounded.  Each operation on them rounds on its own (no contraction), so that the codes can be
// reproduced by any fp32 arithmetic; the update's square root and quotient are the hardware's (1 ulp each).
__device__ __forceinline__ void update(float& p, float g, float& m, float& v, const Coef& k, float step_size, float inv_bc2_sqrt) {
#pragma clang fp contract(off)
  g = g * k.clip;
  m = m + k.one_m_b1 * (g - m);
  v = k.b2 * v + k.one_m_b2 * g * g;
  const bool tiny = v < 0x1p-96f;
  const float root = __builtin_amdgcn_sqrtf(tiny ? v * 0x1p64f : v) * (tiny ? 0x1p-32f : 1.0f);
  p = p * k.decay - step_size * (m * __builtin_amdgcn_rcpf(root * inv_bc2_sqrt + k.eps));
}

// maximum over the wavefront: two half swaps and four row rotations, no LDS
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(b[0], b[1]);
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x128, 0xf, 0xf, false));   // row_ror:8
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x124, 0xf, 0xf, false));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x122, 0xf, 0xf, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x121, 0xf, 0xf, false));
}

__global__ __launch_bounds__(kThreads) void k_adamw8(float* __restrict__ p, const float* __restrict__ g, uint8_t* __restrict__ m,
                                                     uint8_t* __restrict__ v, uint8_t* __restrict__ m_exp, uint8_t* __restrict__ v_exp,
                                                     const int64_t* __restrict__ chunk_off, const int32_t* __restrict__ chunk_len,
                                                     const int32_t* __restrict__ chunk_param, const uint8_t* __restrict__ active,
                                                     int64_t n_chunks, double* __restrict__ hyper, float* __restrict__ pstep,
                                                     const uint32_t* __restrict__ seed, const float* __restrict__ ws, int n_ws,
                                                     const ChunkCoef* __restrict__ coef) {
  __shared__ double shd[kWaves];
  __shared__ Coef shk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double acc = 0.0;
  for (int i = threadIdx.x; i < n_ws; i += kThreads) acc += (double)ws[i];
  for (int o = 32; o; o >>= 1) acc += __shfl_xor(acc, o);
  if (lane == 0) shd[wave] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(shd[0] + shd[1] + shd[2] + shd[3]);
    const float most = (float)hyper[H_MAXNORM];
    Coef k;
    k.decay = (float)(1.0 - hyper[H_LR] * hyper[H_WD]);
    k.one_m_b1 = (float)(1.0 - hyper[H_B1]);
    k.b2 = (float)hyper[H_B2];
    k.one_m_b2 = (float)(1.0 - hyper[H_B2]);
    k.eps = (float)hyper[H_EPS];
    // torch.nn.utils.clip_grad_norm_: max_norm / (total_norm + 1e-6), at most 1
    k.clip = most > 0.f ? fminf(1.0f, most / (norm + 1e-6f)) : 1.0f;
    if (most > 0.f && norm != norm) k.clip = norm;
    shk = k;
    if (blockIdx.x == 0) hyper[H_NORM] = (double)norm;
  }
  __syncthreads();

  const Coef k = shk;
  const uint32_t seed0 = seed[0];
  for (int64_t c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const int prm = chunk_param[c];
    if (!active[prm]) continue;
    const ChunkCoef bc = coef[c];
    if (threadIdx.x == 0 && (c == 0 || chunk_param[c - 1] != prm)) pstep[prm] = bc.step;
    const int64_t off = chunk_off[c];
    const int len = chunk_len[c];
    const uint32_t key = mix32((uint32_t)(int64_t)bc.step * 0x9E3779B9u + seed0);
    const bool wide = ((reinterpret_cast<uintptr_t>(p + off) | reinterpret_cast<uintptr_t>(g + off)) & 15) == 0 &&
                      ((reinterpret_cast<uintptr_t>(m + off) | reinterpret_cast<uintptr_t>(v + off)) & 3) == 0;
    for (int b = wave; b * kBlock < len; b += kWaves) {
      const int i0 = b * kBlock + lane * 4;
      const int64_t at = off + i0;
      const int n = min(4, len - i0);   // <= 0: nothing for this lane
      float P[4] = {0.f, 0.f, 0.f, 0.f}, G[4] = {0.f, 0.f, 0.f, 0.f}, M[4], V[4];
      uint32_t cm = 0, cv = 0;
      const bool full = wide && n == 4;
      if (full) {
        const float4 x = *reinterpret_cast<const float4*>(p + at), y = *reinterpret_cast<const float4*>(g + at);
        P[0] = x.x; P[1] = x.y; P[2] = x.z; P[3] = x.w;
        G[0] = y.x; G[1] = y.y; G[2] = y.z; G[3] = y.w;
        cm = *reinterpret_cast<const uint32_t*>(m + at);
        cv = *reinterpret_cast<const uint32_t*>(v + at);
      } else {
        for (int i = 0; i < 4; ++i)
          if (i < n) {
            P[i] = p[at + i];
            G[i] = g[at + i];
            cm |= (uint32_t)m[at + i] << (8 * i);
            cv |= (uint32_t)v[at + i] << (8 * i);
          }
      }
      const float um = unit_of(m_exp[c * kPer + b]), uv = unit_of(v_exp[c * kPer + b]);
      uint32_t tm = 0, tv = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = (cm >> (8 * i)) & 255u, y = (cv >> (8 * i)) & 255u;
        const float s = units_of(x & 127u) * um;
        M[i] = x & 128u ? -s : s;
        V[i] = units_of(y) * uv;
        update(P[i], G[i], M[i], V[i], k, bc.size, bc.inv_bc2_sqrt);
        if (i < n) {
          tm = max(tm, __float_as_uint(M[i]) & 0x7fffffffu);
          tv = max(tv, __float_as_uint(V[i]) & 0x7fffffffu);
        }
      }
      tm = wave_max(tm);
      tv = wave_max(tv);
      const int em = unit_exponent(tm, 18), ev = unit_exponent(tv, 34);
      const float im = unit_of(254 - (em == 255 ? 0 : em)), iv = unit_of(254 - (ev == 255 ? 0 : ev));   // 2^-k
      cm = cv = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t idx = (uint64_t)(at + i);
        const uint32_t r = mix32((uint32_t)idx + key + (uint32_t)(idx >> 32) * 0x85EBCA6Bu);
        uint32_t x = 0, y = 0;
        if (em != 0 && em != 255) {
          x = code_of(fabsf(M[i]) * im, r & 0xffffu);
          x |= M[i] < 0.f && x ? 128u : 0u;
        }
        if (ev != 0 && ev != 255) {
          y = code_of(V[i] * iv, r >> 16);
          if (y == 0 && V[i] > 0.f) y = 1;
        }
        cm |= x << (8 * i);
        cv |= y << (8 * i);
      }
      if (full) {
        *reinterpret_cast<float4*>(p + at) = make_float4(P[0], P[1], P[2], P[3]);
        *reinterpret_cast<uint32_t*>(m + at) = cm;
        *reinterpret_cast<uint32_t*>(v + at) = cv;
      } else {
        for (int i = 0; i < 4; ++i)
          if (i < n) {
            p[at + i] = P[i];
            m[at + i] = (uint8_t)(cm >> (8 * i));
            v[at + i] = (uint8_t)(cv >> (8 * i));
          }
      }
      if (lane == 0) {
        m_exp[c * kPer + b] = (uint8_t)em;
        v_exp[c * kPer + b] = (uint8_t)ev;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_adamw8_values(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                            const uint8_t* __restrict__ m_exp, const uint8_t* __restrict__ v_exp,
                                                            const int64_t* __restrict__ chunk_off, const int32_t* __restrict__ chunk_len,
                                                            int64_t n_chunks, const int64_t* __restrict__ gap_off,
                                                            const int32_t* __restrict__ gap_len, T* __restrict__ mo, T* __restrict__ vo) {
  const int64_t c = blockIdx.x;
  if (c >= n_chunks) {
    const int64_t off = gap_off[c - n_chunks];
    for (int i = threadIdx.x; i < gap_len[c - n_chunks]; i += kThreads) {
      if (mo) mo[off + i] = (T)0.f;
      if (vo) vo[off + i] = (T)0.f;
    }
    return;
  }
  const int64_t off = chunk_off[c];
  const int len = chunk_len[c];
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const bool wide = (off & 3) == 0 && ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3) == 0 &&
                    ((reinterpret_cast<uintptr_t>(mo) | reinterpret_cast<uintptr_t>(vo)) & 15) == 0;
  for (int i0 = threadIdx.x * 4; i0 < len; i0 += kThreads * 4) {
    const int b = i0 / kBlock, n = min(4, len - i0);
    const float um = unit_of(m_exp[c * kPer + b]), uv = unit_of(v_exp[c * kPer + b]);
    const bool full = wide && n == 4;
    uint32_t cm = 0, cv = 0;
    if (full) {
      cm = *reinterpret_cast<const uint32_t*>(m + off + i0);
      cv = *reinterpret_cast<const uint32_t*>(v + off + i0);
    } else {
      for (int i = 0; i < n; ++i) {
        cm |= (uint32_t)m[off + i0 + i] << (8 * i);
        cv |= (uint32_t)v[off + i0 + i] << (8 * i);
      }
    }
    vec4 M, V;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = (cm >> (8 * i)) & 255u;
      const float s = units_of(x & 127u) * um;
      M[i] = (T)(x & 128u ? -s : s);
      V[i] = (T)(units_of((cv >> (8 * i)) & 255u) * uv);
    }
    if (full) {
      if (mo) *reinterpret_cast<vec4*>(mo + off + i0) = M;
      if (vo) *reinterpret_cast<vec4*>(vo + off + i0) = V;
    } else {
      for (int i = 0; i < n; ++i) {
        if (mo) mo[off + i0 + i] = M[i];
        if (vo) vo[off + i0 + i] = V[i];
      }
    }
  }
}

int norm_blocks(int64_t n_chunks) { return (int)(n_chunks < kNormBlocks ? n_chunks : kNormBlocks); }

}  // namespace

extern "C" {

int gps_adamw8_block(void) { return kBlock; }

size_t gps_adamw8_workspace_floats(int64_t n_chunks) { return n_chunks > 0 ? (size_t)norm_blocks(n_chunks) + 3 * (size_t)n_chunks : 0; }

int gps_adamw8_step(float* p, const float* g, uint8_t* m, uint8_t* v, uint8_t* m_exp, uint8_t* v_exp, const int64_t* chunk_off,
                    const int32_t* chunk_len, const int32_t* chunk_param, const uint8_t* active, int64_t n_chunks, double* hyper,
                    float* pstep, const uint32_t* seed, float* ws, gps_stream_t stream) {
  GPS_REQUIRE(n_chunks >= 0 && n_chunks < (int64_t(1) << 31), "gps_adamw8_step: n_chunks=%lld", (long long)n_chunks);
  if (n_chunks == 0) return GPS_OK;
  GPS_REQUIRE(p && g && m && v && m_exp && v_exp && chunk_off && chunk_len && chunk_param && active && hyper && pstep && seed && ws,
              "gps_adamw8_step: null pointer argument");
  GPS_REQUIRE(gps_optim_chunk() == kChunk, "gps_adamw8_step: chunk table of %d elements", gps_optim_chunk());
  hipStream_t s = gps::as_stream(stream);
  const int nb = norm_blocks(n_chunks);
  ChunkCoef* coef = reinterpret_cast<ChunkCoef*>(ws + nb);
  k_sqnorm8<<<nb, kThreads, 0, s>>>(g, chunk_off, chunk_len, chunk_param, active, n_chunks, hyper, pstep, ws, coef);
  k_adamw8<<<(unsigned)(n_chunks < kStepBlocks ? n_chunks : kStepBlocks), kThreads, 0, s>>>(
      p, g, m, v, m_exp, v_exp, chunk_off, chunk_len, chunk_param, active, n_chunks, hyper, pstep, seed, ws, nb, coef);
  return gps::launch_status("gps_adamw8_step");
}

int gps_adamw8_values(const uint8_t* m, const uint8_t* v, const uint8_t* m_exp, const uint8_t* v_exp, const int64_t* chunk_off,
                      const int32_t* chunk_len, int64_t n_chunks, const int64_t* gap_off, const int32_t* gap_len, int64_t n_gaps,
                      int dtype, void* m_out, void* v_out, gps_stream_t stream) {
  GPS_REQUIRE(n_chunks >= 0 && n_gaps >= 0 && n_chunks + n_gaps < (int64_t(1) << 31), "gps_adamw8_values: %lld chunks, %lld gaps",
              (long long)n_chunks, (long long)n_gaps);
  GPS_REQUIRE(dtype == GPS_F32 || dtype == GPS_BF16, "gps_adamw8_values: dtype %d", dtype);
  if (n_chunks + n_gaps == 0) return GPS_OK;
  GPS_REQUIRE(n_chunks == 0 || (m && v && m_exp && v_exp && chunk_off && chunk_len), "gps_adamw8_values: null pointer argument");
  GPS_REQUIRE(n_gaps == 0 || (gap_off && gap_len), "gps_adamw8_values: null pointer argument");
  hipStream_t s = gps::as_stream(stream);
  const unsigned grid = (unsigned)(n_chunks + n_gaps);
  if (dtype == GPS_F32)
    k_adamw8_values<float><<<grid, kThreads, 0, s>>>(m, v, m_exp, v_exp, chunk_off, chunk_len, n_chunks, gap_off, gap_len,
                                                     static_cast<float*>(m_out), static_cast<float*>(v_out));
  else
    k_adamw8_values<__bf16><<<grid, kThreads, 0, s>>>(m, v, m_exp, v_exp, chunk_off, chunk_len, n_chunks, gap_off, gap_len,
                                                      static_cast<__bf16*>(m_out), static_cast<__bf16*>(v_out));
  return gps::launch_status("gps_adamw8_values");
}

}  // extern "C"
