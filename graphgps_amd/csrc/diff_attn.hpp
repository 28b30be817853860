// Differential attention: shared pieces of its kernels (diff_attn.hip, diff_attn_bwd.hip).  gfx950 only.
//
//   o = (softmax(s q1 k1^T) - lam softmax(s q2 k2^T)) v        per segment and head; d columns per map, 2d columns of v
//
// Everything is written on 16 x 16 matrix-instruction tiles with a contraction of 32 and ONE fragment layout: lane l holds
// eight elements of row (A) or column (B) l & 15, the contraction slots (l >> 4) * 8 + j.  16-bit types take one
// v_mfma_f32_16x16x32; fp32 takes eight v_mfma_f32_16x16x4_f32, the j-th on element j of every lane (a contraction may be
// summed in any order as long as both operands agree on it), so fp32 inputs keep fp32 products.
// A result tile has column l & 15 and rows (l >> 4) * 4 + r in register r.  Two result tiles of one column block, converted,
// ARE a B fragment over their 32 rows if slot (g, j) is read as row g * 4 + j (j < 4) or 16 + g * 4 + j - 4: attention
// weights feed the next product from the registers they were computed in.  The other operand of that product is then a
// matrix read down its columns: ds_read_b64_tr_b16 hands lane l the four elements (g * 4 .. g * 4 + 3, l & 15) of a row-major
// LDS tile, which is that slot order.
#pragma once
#include "gps_common.hpp"

namespace diffattn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kInf = __builtin_huge_valf();
constexpr float kLowest = 3.4028234e38f;   // -kLowest: the reference of a row that has seen nothing (finite: -inf scores stay weight 0)

using Args = gps_diff_attn;   // include/gps_hip.h

template <typename T>
struct Frag {
  vec_t<T, 8> v;
};
template <>
struct Frag<float> {
  f32x4 lo, hi;
};

__device__ __forceinline__ f32x4 mma(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<f16>& a, const Frag<f16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[j], b.lo[j], c, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[j], b.hi[j], c, 0, 0, 0);
  return c;
}

// eight contiguous elements at p (16-byte aligned; global or LDS)
template <typename T>
__device__ __forceinline__ Frag<T> frag_load(const T* p) {
  Frag<T> f;
  if constexpr (sizeof(T) == 4) {
    f.lo = *reinterpret_cast<const f32x4*>(p);
    f.hi = *reinterpret_cast<const f32x4*>(p + 4);
  } else {
    f.v = *reinterpret_cast<const vec_t<T, 8>*>(p);
  }
  return f;
}
template <typename T>
__device__ __forceinline__ Frag<T> frag_zero() {
  Frag<T> f;
  if constexpr (sizeof(T) == 4) {
    f.lo = f32x4{0.f, 0.f, 0.f, 0.f};
    f.hi = f.lo;
  } else {
    f.v = vec_t<T, 8>(0);
  }
  return f;
}
// two result tiles -> the B fragment over their 32 rows.  16-bit types round to nearest here: the weights and their
// gradients enter the second product in the input's type, which is what the matrix instruction takes; frag_lost makes a second
// operand of what that rounding lost.
template <typename T>
__device__ __forceinline__ Frag<T> frag_pack(f32x4 a, f32x4 b) {
  Frag<T> f;
  if constexpr (sizeof(T) == 4) {
    f.lo = a;
    f.hi = b;
  } else {
    const vec_t<T, 4> x = __builtin_convertvector(a, vec_t<T, 4>), y = __builtin_convertvector(b, vec_t<T, 4>);
    f.v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}
// what frag_pack lost, as a fragment of its own (16-bit types).  The two bfloat16 of a packed register are widened by a shift and a mask:
// left to the compiler, each value is converted a second time first.
__device__ __forceinline__ Frag<bf16> frag_lost(f32x4 a, f32x4 b, const Frag<bf16>& f) {
  const vec_t<uint32_t, 4> w = __builtin_bit_cast(vec_t<uint32_t, 4>, f.v);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    a[2 * j] -= __uint_as_float(w[j] << 16);
    a[2 * j + 1] -= __uint_as_float(w[j] & 0xffff0000u);
    b[2 * j] -= __uint_as_float(w[2 + j] << 16);
    b[2 * j + 1] -= __uint_as_float(w[2 + j] & 0xffff0000u);
  }
  return frag_pack<bf16>(a, b);
}
__device__ __forceinline__ Frag<f16> frag_lost(f32x4 a, f32x4 b, const Frag<f16>& f) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] -= (float)f.v[j];
    b[j] -= (float)f.v[4 + j];
  }
  return frag_pack<f16>(a, b);
}
// A fragment of the TRANSPOSE of the row-major LDS tile `m` (row stride `ld`): row of A = column col0 + (l & 15), slots = rows
// row0 .. row0 + 31 in frag_pack's order
template <typename T>
__device__ __forceinline__ Frag<T> frag_tr(const T* m, int ld, int row0, int col0, int lane) {
  Frag<T> f;
  const int g = lane >> 4, i = lane & 15;
  if constexpr (sizeof(T) == 4) {
    const float* p = m + (row0 + g * 4) * ld + col0 + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f.lo[j] = p[j * ld];
      f.hi[j] = p[(16 + j) * ld];
    }
  } else {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    T* p = const_cast<T*>(m) + (row0 + g * 4 + (i >> 2)) * ld + col0 + (i & 3) * 4;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * ld));
    f.v = __builtin_bit_cast(vec_t<T, 8>, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  return f;
}

// IEEE maximum (a NaN stays one): one instruction, where fmaxf first makes its operands canonical
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// op over the four lane groups (same lane & 15); every lane gets it
template <typename Op>
__device__ __forceinline__ float over_groups(float x, Op op) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// four results -> four contiguous elements of T at p (aligned to four elements)
template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 x) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<f32x4*>(p) = x;
  else
    *reinterpret_cast<vec_t<T, 4>*>(p) = __builtin_convertvector(x, vec_t<T, 4>);
}

// the output's four elements from `at` on, and what they lose by rounding: dO . o over a row of o enters every dS of that row, so an
// o that is rounded there would leave its error in all of them (rows that see a few keys: as large as what is left of dS)
template <typename T>
__device__ __forceinline__ void store_out4(const Args& a, int64_t at, f32x4 x) {
  store4(static_cast<T*>(a.o) + at, x);
  if constexpr (sizeof(T) == 2)
    if (a.o_rest) store4(static_cast<T*>(a.o_rest) + at, x - __builtin_convertvector(__builtin_convertvector(x, vec_t<T, 4>), f32x4));
}

__device__ __forceinline__ float load_lam(const Args& a, int h, const bf16*) {
  return a.lam_f32 ? static_cast<const float*>(a.lam)[h] : (float)static_cast<const bf16*>(a.lam)[h];
}
__device__ __forceinline__ float load_lam(const Args& a, int h, const f16*) {
  return a.lam_f32 ? static_cast<const float*>(a.lam)[h] : (float)static_cast<const f16*>(a.lam)[h];
}
__device__ __forceinline__ float load_lam(const Args& a, int h, const float*) { return static_cast<const float*>(a.lam)[h]; }

__device__ __forceinline__ int clamp_row(int32_t r, int64_t n) { return r < 0 ? 0 : (r > n ? (int)n : r); }

// Which rows tile `tile` covers (find_tile below), without a tile map and without the host knowing the segment lengths.  Segment s owns the tile
// numbers from ptr[s] / bm + s on: that grows by at least ceil(length / bm) from each segment to the next and never passes
// N / bm + B, so N / bm + B + 1 tiles cover every segment and the rows behind the last one (segment B).  64 lanes probe at a
// time: two rounds for up to 4,096 segments.  Lane-uniform.  Entries outside [0, N] are cut to it: no row index leaves N.
//
// Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own: workgroup b of `tiles` x `heads` takes a unit such
// that an XCD works on as few heads as possible (all tiles of a head read the same rows), with neighbouring tiles spread over the
// XCDs that share a head (they are unequal where segments are, or under a causal mask).  Grid: xcd_grid(tiles * heads).  Forward of two
// graphs of ~4,700 nodes, 8 heads of 64 columns: 386-392 us, 418 with heads in turn; the backward is the same with either.
struct Unit {
  int tile, head;
};
__device__ __forceinline__ Unit xcd_unit(int b, int tiles, int heads) {
  const int x = b & 7, i = b >> 3;
  if (8 % heads == 0) return {i * (8 / heads) + x / heads, x % heads};
  if (heads % 8 == 0) return {i % tiles, x + 8 * (i / tiles)};
  return {b % tiles, b / tiles};
}
__host__ __device__ __forceinline__ int xcd_grid(int units) { return (units + 7) / 8 * 8; }

template <typename In>
__device__ __forceinline__ int last_segment(int B, In in) {   // the last s in 0 .. B with in(s); in(0) holds, and in() only ends once
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = B;
  while (lo < hi) {
    const int step = (hi - lo + 63) >> 6;
    const int s = lo + (lane + 1) * step;
    const int n = __popcll(__ballot(s <= hi && in(s)));
    lo += n * step;
    hi = min(hi, lo + step - 1);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}
__device__ __forceinline__ int find_segment(const int32_t* ptr, int B, int64_t N, int64_t row) {
  return last_segment(B, [&](int s) { return clamp_row(ptr[s], N) <= row; });
}

struct Tile {
  int seg, first, rows;  // segment (B = behind the last one), first row, rows in this tile (<= 0: none)
  int local;             // index of `first` in the segment
  int len;               // rows of the segment
};
__device__ __forceinline__ Tile find_tile(const int32_t* ptr, int B, int64_t N, int bm, int tile) {
  Tile t;
  t.seg = last_segment(B, [&](int s) { return clamp_row(ptr[s], N) / bm + s <= tile; });
  const int begin = clamp_row(ptr[t.seg], N);
  const int end = t.seg < B ? clamp_row(ptr[t.seg + 1], N) : (int)N;
  t.local = (tile - (begin / bm + t.seg)) * bm;
  t.first = begin + t.local;
  t.rows = t.local < 0 ? 0 : min(bm, end - t.first);
  t.len = max(0, end - begin);
  return t;
}

// --- LDS tiles: R rows of C elements, no padding, 16-byte chunks of a row permuted by its number (chunk c of row r sits at place
// c ^ swz(r)).  Loads can then go straight from memory to LDS (a wavefront's load fills 1 KB of consecutive LDS, each lane picking its
// own address in memory), and both readers below touch every bank equally often.
template <typename T, int C>
struct Tl {
  static constexpr int El = 16 / sizeof(T), CH = C / El, RB = C * sizeof(T);   // elements per chunk, chunks and bytes per row
  static_assert((CH & (CH - 1)) == 0 && RB >= 64, "power of two rows");
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (RB >= 256)
      return r & 15;
    else
      return (r / (256 / RB)) & (CH - 1);
  }
  static __device__ __forceinline__ int at(int r, int chunk) { return r * C + ((chunk ^ swz(r)) * El); }

  // A / B fragment: eight elements from column c (a multiple of 8) of row r
  static __device__ __forceinline__ Frag<T> frag(const T* m, int r, int c) {
    Frag<T> f;
    if constexpr (sizeof(T) == 4) {
      f.lo = *reinterpret_cast<const f32x4*>(m + at(r, c / 4));
      f.hi = *reinterpret_cast<const f32x4*>(m + at(r, c / 4 + 1));
    } else {
      f.v = *reinterpret_cast<const vec_t<T, 8>*>(m + at(r, c / 8));
    }
    return f;
  }
  // A fragment of the transpose: row of A = column col0 + (l & 15), slots = rows row0 .. row0 + 31 in frag_pack's order
  static __device__ __forceinline__ Frag<T> frag_tr(const T* m, int row0, int col0, int lane) {
    Frag<T> f;
    const int g = lane >> 4, i = lane & 15;
    if constexpr (sizeof(T) == 4) {
      const int c = col0 + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = row0 + g * 4 + j;
        f.lo[j] = m[at(r, c >> 2) + (c & 3)];
        f.hi[j] = m[at(r + 16, c >> 2) + (c & 3)];
      }
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const int r = row0 + g * 4 + (i >> 2), c = col0 + (i & 3) * 4;
      T* p = const_cast<T*>(m) + at(r, c >> 3) + (c & 7);   // swz(r + 16) = swz(r)
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * C));
      f.v = __builtin_bit_cast(vec_t<T, 8>, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return f;
  }
};

// R rows into the tile `dst` straight from memory (complete after the next wait for vector memory).  The C columns are Maps
// equal parts, `map_stride` apart in memory, of which `cols` elements exist each.  Rows at and past n (n >= 1) repeat row n - 1 and
// columns past `cols` repeat the last chunk: they meet weights or operands that are zero, and bring nothing a real key does not.
template <typename T, int R, int C, int Maps>
__device__ __forceinline__ void stage_async(T* dst, const T* src, int64_t row_stride, int64_t map_stride, int n, int cols) {
  typedef Tl<T, C> L;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  for (int i = wave; i < R * L::CH / 64; i += waves) {
    const int x = i * 64 + lane, r = x / L::CH, chunk = (x % L::CH) ^ L::swz(r);
    const int m = chunk / (L::CH / Maps), c = min(chunk % (L::CH / Maps) * L::El, cols - L::El);
    const T* p = src + (int64_t)min(r, n - 1) * row_stride + (Maps > 1 ? m * map_stride : 0) + c;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                     (__attribute__((address_space(3))) void*)(dst + i * 64 * L::El), 16, 0, 0);
  }
}
// The same for workgroups of 256 threads with the lanes' offsets from a tile's first row worked out once: what is left per block is
// one uniform address.  Tiles that are not full, and smaller workgroups, go through stage_async.
template <typename T, int R, int C, int Maps>
struct Stager {
  typedef Tl<T, C> L;
  static constexpr int Loads = R * L::CH / 256;
  uint32_t off[Loads];
  __device__ __forceinline__ Stager(int64_t row_stride, int64_t map_stride, int cols) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < Loads; ++j) {
      const int x = (j * 4 + wave) * 64 + lane, r = x / L::CH, chunk = (x % L::CH) ^ L::swz(r);
      const int m = chunk / (L::CH / Maps), c = min(chunk % (L::CH / Maps) * L::El, cols - L::El);
      off[j] = (uint32_t)((r * row_stride + (Maps > 1 ? m * map_stride : 0) + c) * (int64_t)sizeof(T));
    }
  }
  __device__ __forceinline__ void operator()(T* dst, const T* src, int64_t row_stride, int64_t map_stride, int n, int cols) const {
    if (n == R && blockDim.x == 256) {
      const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
      for (int j = 0; j < Loads; ++j)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(reinterpret_cast<const char*>(src) + off[j]),
                                         (__attribute__((address_space(3))) void*)(dst + (j * 4 + wave) * 64 * L::El), 16, 0, 0);
    } else {
      stage_async<T, R, C, Maps>(dst, src, row_stride, map_stride, n, cols);
    }
  }
};
// This thread's row of a tile of R rows, and its part in zeroing it: 0 * NaN is not 0, so rows that the contraction meets with a
// weight of zero must not hold whatever a dropped row holds.  blockDim.x / R threads (one at least) share a row.
template <int R>
struct RowShare {
  int per, row, part;
  __device__ __forceinline__ RowShare() : per(blockDim.x / R), row(threadIdx.x / (blockDim.x / R)), part(threadIdx.x % (blockDim.x / R)) {}
  template <typename T, int C>
  __device__ __forceinline__ void zero(T* tile) const {
    for (int c = part; c < Tl<T, C>::CH; c += per) *reinterpret_cast<uint4*>(tile + row * C + c * Tl<T, C>::El) = make_uint4(0, 0, 0, 0);
  }
};
// this wavefront's loads into LDS have arrived, and everybody's have: tiles written before are readable, tiles read before are free
__device__ __forceinline__ void tiles_ready() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

template <typename T>
void backward(const Args& a, hipStream_t s);   // diff_attn_bwd.hip

// diff_attn_few.hip: few queries over many keys
bool few_applies(const Args& a);
size_t few_workspace_floats(const Args& a);
template <typename T>
void forward_few(const Args& a, hipStream_t s);

}  // namespace diffattn
