// Dense layers in 8-bit floating point for MI355X (gfx950, CDNA4).
//
// Numbers. A block of 128 values shares one power of two s = 2^e, the
// smallest with max|v| <= 448 s (e >= -126), and each value is stored as
// e4m3(v / s), rounded to nearest, ties to even. s is stored as the byte
// e + 127. A power of two divides exactly, so the one rounding is e4m3's
// (half a step is 2^-4 of the value), and the matrix instruction takes the
// byte as it is: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128-long
// rows, scales each product of blocks and adds in 32 bits, so that a block
// of 128 costs no vector instruction at all. Values that are not finite are
// stored as e4m3's NaN and leave their block's scale alone.
//
// Two ways to multiply. The 8-bit matrix instructions of this chip add eight
// neighbouring products with about 16 bits below the largest of them (32
// only between such groups): 1.6e-5 of a result's norm, measured over random
// e4m3. That is far below e4m3's and a 16-bit result's own rounding, but not
// 32 bits. So where a result is returned in 32 bits, or the sign of a sum
// decides a relu's gradient, the bytes are widened to bf16 in registers on the
// way (exactly, scale included, from 2^-133 up) and multiplied by the bf16
// instruction, whose sums hold 24 bits (8e-9 measured), at half the rate. The
// error of a sum is in proportion to its largest products, not to its own size
// or its neighbours', so a result says nothing of how near to zero is too
// near, and all of a relu's sums are taken in 32 bits.
//
// Layout. A matrix [R, C] that is contracted over C is stored as bytes
// [R, Cp], Cp = C rounded up to 128 (zeros behind C), with scales
// [Cp/128, Rp], Rp = R rounded up to 256. Within each 64 rows the scale
// bytes are permuted (scale_slot below) so that a lane finds the bytes of
// the four fragments that it multiplies in one 32-bit word.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fp8_kernels.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
typedef __attribute__((ext_vector_type(2))) short s16x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

namespace {

constexpr int kBlk = EDL_FP8_BLOCK;

// ------------------------------ small pieces ------------------------------
__device__ inline float as_f32(float v) { return v; }
__device__ inline float as_f32(__bf16 v) { return (float)v; }
__device__ inline float as_f32(_Float16 v) { return (float)v; }

__device__ inline float load_any(const void* p, int64_t i, int type) {
  if (type == EDL_T_F32) return static_cast<const float*>(p)[i];
  if (type == EDL_T_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}

__device__ inline void store_any(void* p, int64_t i, float v, int type) {
  if (type == EDL_T_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == EDL_T_BF16)
    static_cast<__bf16*>(p)[i] = (__bf16)v;
  else
    static_cast<_Float16*>(p)[i] = (_Float16)v;
}

__device__ inline float activate(float z, int act) {
  if (act == EDL_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
  if (act == EDL_ACT_SIGMOID) return 1.f / (1.f + __expf(-z));
  return z;
}

// |v|'s bits, 0 where v is infinite or NaN; as integers they order like |v|
__device__ inline uint32_t finite_abs(float v) {
  uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// The byte e + 127 of the smallest 2^e with amax <= 448 * 2^e:
// 448 = 1.75 * 2^8, so e is amax's exponent - 8, and one more where amax's
// mantissa is over 1.75. At least 1 (2^-126), so that 2^-e is normal.
__device__ inline int scale_byte(uint32_t amax) {
  int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < 1 ? 1 : b;
}

__device__ inline float inverse_of(int byte) {  // 2^(127 - byte), exact
  return __uint_as_float((uint32_t)(254 - byte) << 23);
}

// x / s, and NaN where x is not finite (infinity * 0), which the conversion
// stores as 0xff; it would take infinity for a large number
__device__ inline float scaled(float x, float inv) {
  return __builtin_fmaf(x, 0.f, x * inv);
}

__device__ inline uint32_t pack4(float a, float b, float c, float d,
                                 float inv) {
  int v = 0;
  v = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(a, inv), scaled(b, inv), v, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(c, inv), scaled(d, inv), v, true);
  return (uint32_t)v;
}

// where row r's scale byte lies within its column of Rp bytes
__device__ inline int64_t scale_slot(int64_t r) {
  int n = (int)(r & 63);
  return (r & ~(int64_t)63) + (n >> 4) * 16 + (n & 3) * 4 + ((n >> 2) & 3);
}

// largest over the 16 lanes of a row of lanes
template <int CTRL>
__device__ inline uint32_t max_ror(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf,
                                                     false);
  return v > o ? v : o;
}
__device__ inline uint32_t max16(uint32_t v) {
  v = max_ror<0x128>(v);  // row_ror:8, 4, 2, 1
  v = max_ror<0x124>(v);
  v = max_ror<0x122>(v);
  return max_ror<0x121>(v);
}

// --------------------------------- quantise -------------------------------
// One workgroup takes a tile of 128 x 128 and each thread ROWS x 8 of it, so
// that a block's maximum lies in one 16-lane row of lanes (rows) or in the
// waves (columns), and both forms are written from one read of x. Bound by
// memory where there are many tiles (8 rows to a thread: 16384 x 4096 76 us,
// against 85 with 4), by a thread's work where there are few (4096 x 624 10.2
// us with 4, 12.8 with 8).
//
// DERIV: x is the gradient at an activation's output, which is turned into
// the gradient at its input on the way (relu: one kept bit; sigmoid: the
// kept output), and its column sums are the bias's gradient.
template <typename T>
__device__ inline void load8(const T* p, float* v);
template <>
__device__ inline void load8<float>(const float* p, float* v) {
  f32x4 a = *reinterpret_cast<const f32x4*>(p);
  f32x4 b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    v[c] = a[c];
    v[4 + c] = b[c];
  }
}
template <>
__device__ inline void load8<__bf16>(const __bf16* p, float* v) {
  bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int c = 0; c < 8; ++c) v[c] = (float)a[c];
}
template <>
__device__ inline void load8<_Float16>(const _Float16* p, float* v) {
  f16x8 a = *reinterpret_cast<const f16x8*>(p);
#pragma unroll
  for (int c = 0; c < 8; ++c) v[c] = (float)a[c];
}

// 8 values of row r from column c; zeros outside the matrix
template <typename T>
__device__ inline void load_row8(const T* x, int64_t ld, int64_t R, int64_t C,
                                 int64_t r, int64_t c, bool wide, float* v) {
  const T* p = x + r * ld + c;
  if (r < R && c + 8 <= C && wide) {
    load8<T>(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = (r < R && c + k < C) ? as_f32(p[k]) : 0.f;
  }
}

constexpr int kLdsRow = 144;  // a transposed row: 128 bytes and 16 of padding

template <int ROWS>
struct QuantLds {
  static constexpr int kQuantWaves = 32 / ROWS;
  uint32_t max[kQuantWaves][kBlk];
  float sum[kQuantWaves][kBlk];
  __align__(16) uint8_t t[kBlk * kLdsRow];
};

template <typename T, int kQuantRows, bool TILE, bool DERIV>
__device__ inline void quantize_tile(const edl_fp8_quant& a, int64_t block,
                                     QuantLds<kQuantRows>& lds) {
  constexpr int kQuantWaves = QuantLds<kQuantRows>::kQuantWaves;
  uint32_t(*s_max)[kBlk] = lds.max;
  float(*s_sum)[kBlk] = lds.sum;
  uint8_t* s_t = lds.t;
  const bool cols = a.cols != nullptr;  // the transpose too

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int j = tid & 15;  // columns j*8 .. j*8+7
  const int i = tid >> 4;  // rows    i*ROWS ..
  const int64_t ncb = (a.C + kBlk - 1) / kBlk;
  const int64_t rb = block / ncb, cb = block % ncb;
  const int64_t r0 = rb * kBlk + i * kQuantRows, c0 = cb * kBlk + j * 8;

  float v[kQuantRows][8];
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r)
    load_row8<T>(static_cast<const T*>(a.x), a.ld, a.R, a.C, r0 + r, c0,
                 a.wide, v[r]);

  if (DERIV) {
    if (a.act == EDL_ACT_RELU) {
#pragma unroll
      for (int r = 0; r < kQuantRows; ++r) {
        uint32_t bits = 0;
        if (r0 + r < a.R && c0 < a.C)
          bits = a.mask[(r0 + r) * a.mask_ld + (c0 >> 3)];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[r][c] = (bits >> c) & 1 ? v[r][c] : 0.f;
      }
    } else if (a.act == EDL_ACT_SIGMOID) {
#pragma unroll
      for (int r = 0; r < kQuantRows; ++r) {
        float o[8];
        load_row8<T>(static_cast<const T*>(a.y), a.y_ld, a.R, a.C, r0 + r, c0,
                     a.y_wide, o);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[r][c] = v[r][c] * o[c] * (1.f - o[c]);
      }
    }
    if (a.sums) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kQuantRows; ++r) s += v[r][c];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (lane < 16) s_sum[wave][j * 8 + c] = s;
      }
    }
  }

  uint32_t rmax[kQuantRows], cmax[8];
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) rmax[r] = 0;
#pragma unroll
  for (int c = 0; c < 8; ++c) cmax[c] = 0;
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t m = finite_abs(v[r][c]);
      rmax[r] = max(rmax[r], m);
      cmax[c] = max(cmax[c], m);
    }
  if (!TILE) {
#pragma unroll
    for (int r = 0; r < kQuantRows; ++r) rmax[r] = max16(rmax[r]);
  }
  if (cols || TILE) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t m = cmax[c];
      m = max(m, (uint32_t)__shfl_xor((int)m, 16));
      m = max(m, (uint32_t)__shfl_xor((int)m, 32));
      if (lane < 16) s_max[wave][j * 8 + c] = m;
    }
  }
  if (cols || TILE || (DERIV && a.sums)) __syncthreads();

  if (cols || TILE) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      int col = j * 8 + c;
#pragma unroll
      for (int w = 0; w < kQuantWaves; ++w)
        cmax[c] = max(cmax[c], s_max[w][col]);
    }
  }
  if (TILE) {  // one scale for all of it
    uint32_t m = cmax[0];
#pragma unroll
    for (int c = 1; c < 8; ++c) m = max(m, cmax[c]);
    m = max16(m);
#pragma unroll
    for (int r = 0; r < kQuantRows; ++r) rmax[r] = m;
#pragma unroll
    for (int c = 0; c < 8; ++c) cmax[c] = m;
  }
  if (DERIV && a.sums && tid < kBlk) {
    int64_t c = cb * kBlk + tid;
    if (c < a.C)
    {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kQuantWaves; ++w) t += s_sum[w][tid];
      a.sums[rb * a.C + c] = t;
    }
  }

  if (a.rows) {
#pragma unroll
    for (int r = 0; r < kQuantRows; ++r) {
      int b = scale_byte(rmax[r]);
      float inv = inverse_of(b);
      if (j == 0) a.rows_scale[cb * a.rows_rp + scale_slot(r0 + r)] = b;
      if (r0 + r < a.R) {
        i32x2 q;
        q[0] = pack4(v[r][0], v[r][1], v[r][2], v[r][3], inv);
        q[1] = pack4(v[r][4], v[r][5], v[r][6], v[r][7], inv);
        *reinterpret_cast<i32x2*>(a.rows + (r0 + r) * a.rows_ld + c0) = q;
      }
    }
  }
  if (cols) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      int b = scale_byte(cmax[c]);
      float inv = inverse_of(b);
      if (i == 0) a.cols_scale[rb * a.cols_rp + scale_slot(c0 + c)] = b;
      uint8_t* to = s_t + (j * 8 + c) * kLdsRow + i * kQuantRows;
#pragma unroll
      for (int r = 0; r < kQuantRows; r += 4)
        *reinterpret_cast<uint32_t*>(to + r) =
            pack4(v[r][c], v[r + 1][c], v[r + 2][c], v[r + 3][c], inv);
    }
    __syncthreads();
    // 8 lanes write a transposed row's 128 bytes together
#pragma unroll
    for (int s = 0; s < kQuantRows / 2; ++s) {
      int col = s * kQuantWaves * 8 + (tid >> 3), part = (tid & 7) * 16;
      int64_t c = cb * kBlk + col;
      if (c < a.C)
        *reinterpret_cast<i32x4*>(a.cols + c * a.cols_ld + rb * kBlk + part) =
            *reinterpret_cast<const i32x4*>(s_t + col * kLdsRow + part);
    }
  }
}

template <typename T, int ROWS, bool TILE, bool DERIV>
__global__ __launch_bounds__(2048 / ROWS) void quantize_kernel(
    edl_fp8_quant a) {
  __shared__ QuantLds<ROWS> lds;
  quantize_tile<T, ROWS, TILE, DERIV>(a, blockIdx.x, lds);
}

// a layer's input and its weight in one launch
template <typename TX, typename TW, int ROWS>
__global__ __launch_bounds__(2048 / ROWS) void quantize_pair_kernel(
    edl_fp8_quant x, edl_fp8_quant w, int x_tiles) {
  __shared__ QuantLds<ROWS> lds;
  if ((int)blockIdx.x < x_tiles)
    quantize_tile<TX, ROWS, false, false>(x, blockIdx.x, lds);
  else
    quantize_tile<TW, ROWS, true, false>(w, blockIdx.x - x_tiles, lds);
}

// out[c] = sum over the tiles of sums[t][c], in order of t within each of 16
// lanes' share, the shares then in order
__device__ inline void column_sums(const float* __restrict__ sums,
                                   int64_t tiles, int64_t C, void* out,
                                   int type, int64_t block) {
  __shared__ float s[16][17];
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
  const int64_t col = block * 16 + c;
  float t = 0.f;
  if (col < C)
    for (int64_t r = k; r < tiles; r += 16) t += sums[r * C + col];
  s[k][c] = t;
  __syncthreads();
  if (k == 0 && col < C) {
    float u = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) u += s[q][c];
    store_any(out, col, u, type);
  }
}

// --------------------------------- product --------------------------------
// C[m, n] = act(sum over blocks of 128 of sa[m] sb[n] sum_k A[m, k] B[n, k]
//               + bias[n])
//
// A workgroup takes WM*FM*16 x WN*FN*16 of C and a wave FM*16 x FN*16; a
// step is one block of 128. Both tiles pass through two buffers of LDS,
// filled by global_load_lds. A row's 128 bytes are eight 16-byte chunks,
// and chunk c of row r lies at slot c ^ swz(r), which is free of bank
// conflicts both ways.
//
// A fragment's 16 rows are not neighbours: row rr of fragment f is row
// (rr>>2)*16 + f*4 + (rr&3) of its 64. B goes in as the instruction's first
// operand, so that a lane's results are one row of C and, over the four
// fragments, 16 neighbours of it: one or two wide stores, and one 16-bit
// word of the relu mask.
//
// In a step each wave reads its fragments of A two ahead of the
// instructions that use them. Once a wave has read its last fragment and
// the next tile has landed, one barrier hands the buffer over; the
// instructions on the last two fragments cover the first reads of the next
// step.
__device__ inline int swz(int r) { return (r & 3) | ((r >> 2) & 4); }

__device__ inline int xcd_order(int bid, int n) {
  // workgroups go to the 8 XCDs in turn; give each XCD a run of neighbours
  if (n < 8) return bid;
  int xcd = bid & 7, idx = bid >> 3, q = n >> 3, r = n & 7;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

// Memory to LDS without registers: lane l's bytes land at m0 + l * size. The
// address is a buffer's base + the lane's offset + a scalar, so the loop over
// the blocks keeps no 64-bit addresses. Written as assembly because the
// compiler would wait for these loads before any read of LDS that it cannot
// tell from their target, and the two buffers differ at run time only; there
// is no output register, and the loop waits (vmcnt) before each barrier.
__device__ inline i32x4 buffer_of(const uint8_t* p, int64_t bytes) {
  const uint64_t base = (uint64_t)p;
  const int64_t most = 0xffffffffll;
  return (i32x4){(int)(uint32_t)base, (int)(uint32_t)(base >> 32),
                 (int)(uint32_t)(bytes < most ? bytes : most), 0x00027000};
}
__device__ inline void dma16(i32x4 src, uint32_t lane_off, uint32_t off,
                             uint32_t dst) {
  asm volatile(
      "s_mov_b32 m0, %3\n\ts_nop 0\n\t"
      "buffer_load_dwordx4 %1, %0, %2 offen lds" ::"s"(src),
      "v"(lane_off), "s"(off), "s"(dst)
      : "memory", "m0");
}
__device__ inline void dma4(i32x4 src, uint32_t lane_off, uint32_t off,
                            uint32_t dst) {
  asm volatile(
      "s_mov_b32 m0, %3\n\ts_nop 0\n\t"
      "buffer_load_dword %1, %0, %2 offen lds" ::"s"(src),
      "v"(lane_off), "s"(off), "s"(dst)
      : "memory", "m0");
}

template <int OPA, int OPB>
__device__ inline f32x4 mfma(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, OPA,
                                                          sa, OPB, sb);
}
// f: which byte of the scale words; all calls are unrolled to constants
__device__ inline f32x4 mfma_sel(int fa, int fb, i32x8 a, i32x8 b, f32x4 c,
                                 int sa, int sb) {
#define EDL_SEL(X, Y) \
  if (fa == X && fb == Y) return mfma<X, Y>(a, b, c, sa, sb);
  EDL_SEL(0, 0) EDL_SEL(0, 1) EDL_SEL(0, 2) EDL_SEL(0, 3)
  EDL_SEL(1, 0) EDL_SEL(1, 1) EDL_SEL(1, 2) EDL_SEL(1, 3)
  EDL_SEL(2, 0) EDL_SEL(2, 1) EDL_SEL(2, 2) EDL_SEL(2, 3)
  EDL_SEL(3, 0) EDL_SEL(3, 1) EDL_SEL(3, 2)
  return mfma<3, 3>(a, b, c, sa, sb);
#undef EDL_SEL
}

// ---- in 32 bits: a fragment's 32 bytes as four of 8 bf16, times its scale
struct Wide {
  bf16x8 v[4];
};
__device__ inline float scale_value(int word, int f) {
  return __uint_as_float((((uint32_t)word >> (8 * f)) & 0xffu) << 23);
}
__device__ inline Wide widen(i32x8 q, float s) {
  Wide w;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[k], s, false);
    bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[k], s, true);
    const int o = (k & 1) * 4;
    w.v[k >> 1][o] = lo[0];
    w.v[k >> 1][o + 1] = lo[1];
    w.v[k >> 1][o + 2] = hi[0];
    w.v[k >> 1][o + 3] = hi[1];
  }
  return w;
}
__device__ inline f32x4 mfma_wide(const Wide& a, const Wide& b, f32x4 c) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[k], b.v[k], c, 0, 0, 0);
  return c;
}

// results of 32 bits have sums of 32 bits
template <typename T>
constexpr bool is_f32 = sizeof(T) == 4;

__device__ inline void load_bias16(const edl_fp8_gemm& g, int64_t n,
                                   float* bias) {
#pragma unroll
  for (int k = 0; k < 16; ++k)
    bias[k] = g.bias && n + k < g.N ? load_any(g.bias, n + k, g.bias_type)
                                    : 0.f;
}

// 16 neighbours of a row of C, from column n
template <typename T>
__device__ inline void epilogue16(const edl_fp8_gemm& g, int64_t m, int64_t n,
                                  float* v, const float* bias) {
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    v[k] += bias[k];
    bits |= (v[k] > 0.f ? 1u : 0u) << k;
    v[k] = activate(v[k], g.act);
  }
  if (g.mask)
    *reinterpret_cast<uint16_t*>(g.mask + m * g.mask_ld + (n >> 3)) = bits;
  T* p = static_cast<T*>(g.c) + m * g.N + n;
  if (n + 16 <= g.N && g.c_wide) {
    constexpr int W = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
#pragma unroll
    for (int k = 0; k < 16; k += W) {
      vec o;
#pragma unroll
      for (int q = 0; q < W; ++q) o[q] = (T)v[k + q];
      *reinterpret_cast<vec*>(p + k) = o;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (n + k < g.N) p[k] = (T)v[k];
  }
}

// where a workgroup's tile lies, and its share of the steps
struct Spot {
  int64_t m0, n0;
  int split, kb_all, kb0, steps;
};
template <int BM, int BN>
__device__ inline Spot spot_of(const edl_fp8_gemm& g, int block, int blocks) {
  // tiles in groups of 4 rows of tiles, column by column
  const int ntm = (g.M + BM - 1) / BM, ntn = (g.N + BN - 1) / BN;
  const int order = xcd_order(block, blocks);
  const int bid = order % (ntm * ntn);
  const int per = 4 * ntn, grp = bid / per, in = bid % per;
  const int tall = min(4, ntm - grp * 4);
  Spot s;
  s.m0 = (int64_t)(grp * 4 + in % tall) * BM;
  s.n0 = (int64_t)(in / tall) * BN;
  s.split = order / (ntm * ntn);
  s.kb_all = (int)(g.ld / kBlk);
  s.kb0 = (int)((int64_t)s.kb_all * s.split / g.splits);
  s.steps = (int)((int64_t)s.kb_all * (s.split + 1) / g.splits) - s.kb0;
  return s;
}

// A wave's loads of a block: its share of 1 KB pieces of A and of B, each 8
// rows (lane -> row lane>>3, slot lane&7), and 256 bytes of scales, A's by
// even waves and B's by odd ones (several fetch the same; a branch would
// cost more). Rows behind the matrix's last are that one again.
template <int BM, int BN, int NW>
struct Loads {
  static constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;
  static constexpr int kAll = LA + LB + 1;
  i32x4 bufA, bufB, bufS;
  uint32_t offA[LA], offB[LB], offS, at = 0, atS = 0, rp;
  int wave, lane;
  bool odd;

  __device__ Loads(const edl_fp8_gemm& g, const Spot& s, int wave_, int lane_)
      : wave(wave_), lane(lane_), odd(wave_ & 1) {
    const uint8_t* pa = g.a + s.m0 * g.ld + (int64_t)s.kb0 * kBlk;
    const uint8_t* pb = g.b + s.n0 * g.ld + (int64_t)s.kb0 * kBlk;
    bufA = buffer_of(pa, g.a + g.M * g.ld - pa);
    bufB = buffer_of(pb, g.b + g.N * g.ld - pb);
    const uint32_t lastA = (uint32_t)min(g.M - 1 - s.m0, (int64_t)BM);
    const uint32_t lastB = (uint32_t)min(g.N - 1 - s.n0, (int64_t)BN);
#pragma unroll
    for (int q = 0; q < LA; ++q) {
      const uint32_t r = (wave * LA + q) * 8 + (lane >> 3);
      offA[q] = min(r, lastA) * (uint32_t)g.ld + (((lane & 7) ^ swz(r)) << 4);
    }
#pragma unroll
    for (int q = 0; q < LB; ++q) {
      const uint32_t r = (wave * LB + q) * 8 + (lane >> 3);
      offB[q] = min(r, lastB) * (uint32_t)g.ld + (((lane & 7) ^ swz(r)) << 4);
    }
    const int64_t rows = odd ? g.b_rp : g.a_rp;
    const uint8_t* base = odd ? g.sb : g.sa;
    const uint8_t* ps = base + (odd ? s.n0 : s.m0) + s.kb0 * rows;
    bufS = buffer_of(ps, base + (int64_t)s.kb_all * rows - ps);
    rp = (uint32_t)rows;
    // 256 bytes from a tile of fewer rows may be more than there are
    offS = lane * 4;
    if (BM < 256)
      offS = (uint32_t)min((int64_t)offS, rows - 4 - (odd ? s.n0 : s.m0));
  }
  // the q-th load of the next block, into LDS at these places
  __device__ inline void one(uint32_t a, uint32_t b, uint32_t s, int q) {
    if (q < LA) {
      dma16(bufA, offA[q], at, a + (wave * LA + q) * 1024);
    } else if (q < LA + LB) {
      const int o = q - LA;
      dma16(bufB, offB[o], at, b + (wave * LB + o) * 1024);
    } else if (q == LA + LB) {
      dma4(bufS, offS, atS, s + odd * 256);
      at += kBlk;
      atS += rp;
    }
  }
};

// What a wave multiplies: FM fragments of A from the fA0-th, FN of B, and in
// 32 bits (WIDE) B's fragments widened.
//
// Fragment f of the tile's rows: 32 bytes of row rr, in chunks q4 and 4 + q4.
// Which bytes of a block meet is the same for A and B, and a block has one
// scale, so the order within it does not matter. f*4 leaves swz as it is.
template <int FM, int FN, bool WIDE>
struct Hand {
  static constexpr int SA = (FM + 3) / 4;
  static_assert(FN % 4 == 0 && (FM % 4 == 0 || FM == 2), "scale words");
  f32x4 acc[FM][FN];
  i32x8 a[FM], b[FN];
  Wide bw[WIDE ? FN : 1];
  int sa[SA], sb[FN / 4];

  __device__ inline void clear() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int k = 0; k < FN; ++k) acc[i][k] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  static __device__ inline uint32_t row_of(int f) {
    return (f >> 2) * 64 + (f & 3) * 4;
  }
  static __device__ inline i32x8 read(const uint8_t* smem, uint32_t lo,
                                      uint32_t hi, int f) {
    const int o = row_of(f) * kBlk;
    const i32x4 u = *reinterpret_cast<const i32x4*>(smem + lo + o);
    const i32x4 v = *reinterpret_cast<const i32x4*>(smem + hi + o);
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // the words of scales at s: A's from its 64 rows on, shifted to its first
  // fragment; B's 256 bytes behind
  static __device__ inline void read_scales(const uint8_t* s, int fA0, int wB,
                                            int* to_a, int* to_b) {
#pragma unroll
    for (int k = 0; k < SA; ++k) {
      to_a[k] = *reinterpret_cast<const int*>(s + ((fA0 >> 2) + k) * 64);
      if (FM < 4) to_a[k] = (uint32_t)to_a[k] >> ((fA0 & 3) * 8);
    }
#pragma unroll
    for (int k = 0; k < FN / 4; ++k)
      to_b[k] = *reinterpret_cast<const int*>(s + 256 + wB + k * 64);
  }
  __device__ inline void widen_b() {
    if (WIDE) {
#pragma unroll
      for (int k = 0; k < FN; ++k)
        bw[k] = widen(b[k], scale_value(sb[k >> 2], k & 3));
    }
  }
  __device__ inline void product(int i, int k) {
    acc[i][k] = mfma_sel(k & 3, i & 3, b[k], a[i], acc[i][k], sb[k >> 2],
                         sa[i >> 2]);
  }
  __device__ inline void products(int i) {  // fragment i of A, all of B
    if (WIDE) {
      const Wide aw = widen(a[i], scale_value(sa[i >> 2], i & 3));
#pragma unroll
      for (int k = 0; k < FN; ++k) acc[i][k] = mfma_wide(bw[k], aw, acc[i][k]);
    } else {
#pragma unroll
      for (int k = 0; k < FN; ++k) product(i, k);
    }
  }
};

// Lane: row rr of C's 64 and fragment i's 4 i on, columns q4*16 + k*4 + 0..3
// of its 64. The sums pass through LDS, each lane's own, so that one copy of
// the code takes all rows: unrolled, the large tile's 16 would not stay in
// registers.
template <typename T, int FM, int FN, typename H>
__device__ inline void write_tile(const edl_fp8_gemm& g, const Spot& s,
                                  const H& h, uint8_t* smem, int wave,
                                  int lane, int fA0, int wB, bool may_split) {
  constexpr int G = FM < 4 ? FM : 4;
  const int rr = ((lane & 15) >> 2) * 16 + (lane & 3), q4 = lane >> 4;
  f32x4* own = reinterpret_cast<f32x4*>(smem) + wave * (G * 4 * 64) + lane;
  __syncthreads();  // the last blocks are read
#pragma unroll
  for (int p = 0; p < FM / G * (FN / 4); ++p) {  // up to 64 x 64 at a time
    const int j = p % (FN / 4), i0 = p / (FN / 4) * G;
    const int64_t n = s.n0 + wB + j * 64 + q4 * 16;
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        own[(i * 4 + k) * 64] = h.acc[i0 + i][j * 4 + k];
    float bias[16];
    load_bias16(g, n, bias);
#pragma unroll 1
    for (int i = 0; i < G; ++i) {
      const int64_t m = s.m0 + H::row_of(fA0 + i0 + i) + rr;
      const bool live = m < g.M && n < g.N;
      float v[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 u = own[(i * 4 + k) * 64];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[k * 4 + q] = u[q];
      }
      if (may_split && g.splits > 1) {
        float* to = g.part + ((int64_t)s.split * g.M + m) * g.part_ld + n;
        if (live) {
#pragma unroll
          for (int k = 0; k < 16; k += 4)
            *reinterpret_cast<f32x4*>(to + k) =
                (f32x4){v[k], v[k + 1], v[k + 2], v[k + 3]};
        }
      } else {
        if (live) epilogue16<T>(g, m, n, v, bias);
      }
    }
  }
}

template <int BM>
struct GemmLds {  // two buffers each: A's, B's, scales (256 of A's and B's)
  static constexpr uint32_t kTile = BM * kBlk, kB = 2 * kTile, kS = 4 * kTile;
  __align__(1024) uint8_t m[4 * BM * kBlk + 1024];
};

template <int WM, int WN, int FM, int FN, typename T, bool WIDE>
__device__ inline void gemm_tile(const edl_fp8_gemm& g, int block, int blocks,
                                 uint8_t* smem) {
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16, NW = WM * WN;
  static_assert(BM == BN && (BM == 128 || BM == 256), "buffers' toggle");
  constexpr uint32_t kTile = GemmLds<BM>::kTile, kB = GemmLds<BM>::kB,
                     kS = GemmLds<BM>::kS;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const Spot s = spot_of<BM, BN>(g, block, blocks);
  const int steps = s.steps;
  Loads<BM, BN, NW> loads(g, s, wave, lane);
  constexpr int kLoads = Loads<BM, BN, NW>::kAll;
  const uint32_t lds0 =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  auto load = [&](uint32_t buf, int q) {
    loads.one(lds0 + buf * kTile, lds0 + kB + buf * kTile,
              lds0 + kS + buf * 512, q);
  };
  auto stage = [&](uint32_t buf) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) load(buf, q);
  };

  const int rr = ((lane & 15) >> 2) * 16 + (lane & 3), q4 = lane >> 4;
  const uint32_t lo = rr * kBlk + ((q4 ^ swz(rr)) << 4);
  const uint32_t hi = rr * kBlk + (((q4 + 4) ^ swz(rr)) << 4);
  const int wA = wm * FM * 16, wB = wn * FN * 16, fA0 = wm * FM;
  // these move to the other buffer and back with a step
  uint32_t aLo = wA * kBlk + lo, aHi = wA * kBlk + hi;
  uint32_t bLo = kB + wB * kBlk + lo, bHi = kB + wB * kBlk + hi;
  uint32_t sAt = kS + (lane & 15) * 4;
  typedef Hand<FM, FN, WIDE> H;
  H h;
  h.clear();
  int na[FM / 4], nb[FN / 4];
  auto next_scales = [&]() {
#pragma unroll
    for (int k = 0; k < FM / 4; ++k) h.sa[k] = na[k];
#pragma unroll
    for (int k = 0; k < FN / 4; ++k) h.sb[k] = nb[k];
  };

  // Block t + 1 goes into the other buffer in two parts: kEarly loads at the
  // end of step t - 1, behind the barrier that frees it, and the rest (late)
  // between the first products of step t. All at once they would queue up
  // and hold back the reads and products behind them (8192^3: 403 us so, 388
  // in parts).
  constexpr int kEarly = 4;
  constexpr int kLate = (kLoads - kEarly + FM - 3) / (FM - 2) > 2
                            ? (kLoads - kEarly + FM - 3) / (FM - 2)
                            : 2;
  auto step = [&](uint32_t buf, bool late, bool more) {
    h.widen_b();
#pragma unroll
    for (int i = 0; i < FM - 2; ++i) {
      h.a[i + 2] = H::read(smem, aLo, aHi, i + 2);
      h.products(i);
      if (late) {
#pragma unroll
        for (int q = 0; q < kLate; ++q) load(buf ^ 1, kEarly + i * kLate + q);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    aLo ^= kTile;
    aHi ^= kTile;
    bLo ^= kTile;
    bHi ^= kTile;
    sAt ^= 512;
    // after the last step these read a buffer that nobody writes any more
    H::read_scales(smem + sAt, fA0, wB, na, nb);
    h.a[0] = H::read(smem, aLo, aHi, 0);
    h.a[1] = H::read(smem, aLo, aHi, 1);
    __builtin_amdgcn_sched_barrier(0);
    if (WIDE) {
#pragma unroll
      for (int k = 0; k < FN; ++k) h.b[k] = H::read(smem, bLo, bHi, k);
      if (more) {
#pragma unroll
        for (int q = 0; q < kEarly; ++q) load(buf, q);
      }
      __builtin_amdgcn_sched_barrier(0);
      h.products(FM - 2);
      h.products(FM - 1);
    } else {
#pragma unroll
      for (int k = 0; k < FN; ++k) {
        h.product(FM - 2, k);
        h.product(FM - 1, k);
        __builtin_amdgcn_sched_barrier(0);
        h.b[k] = H::read(smem, bLo, bHi, k);
        if (more && k < kEarly) load(buf, k);
      }
    }
    next_scales();
  };

  stage(0);
  if (steps > 1) stage(1);
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  H::read_scales(smem + sAt, fA0, wB, na, nb);
  next_scales();
  h.a[0] = H::read(smem, aLo, aHi, 0);
  h.a[1] = H::read(smem, aLo, aHi, 1);
#pragma unroll
  for (int k = 0; k < FN; ++k) h.b[k] = H::read(smem, bLo, bHi, k);
  // block 1 is there already, and the last steps fetch no more; branches in
  // the loop's body would let the compiler move products behind the barrier
  int t = 0;
  if (steps > 2) {
    step(0, false, true);
    for (t = 1; t + 2 < steps; ++t) step(t & 1, true, true);
    step(t & 1, true, false);
    ++t;
  }
  for (; t < steps; ++t) step(t & 1, false, false);
  write_tile<T, FM, FN>(g, s, h, smem, wave, lane, fA0, wB, BM == 128);
}

template <int WM, int WN, int FM, int FN, typename T, bool WIDE>
__global__ __launch_bounds__(WM* WN * 64, 2) void gemm_kernel(
    edl_fp8_gemm g) {
  __shared__ GemmLds<WM * FM * 16> lds;
  gemm_tile<WM, WN, FM, FN, T, WIDE>(g, blockIdx.x, gridDim.x, lds.m);
}

// Products too small to fill the chip with the tiles above wait for memory,
// not for the matrix cores: a workgroup takes 64 x 128, a wave 32 x 64, and
// the blocks pass through three buffers, so that loads are two steps ahead.
// A step waits for its own block's loads alone (vmcnt counts a wave's, in
// order), then one barrier both shows the block to all waves and frees the
// buffer of the step before, which all have read by then.
struct RingLds {
  static constexpr int BM = 64, BN = 128, kBuffers = 3;
  static constexpr uint32_t kA = BM * kBlk, kB = BN * kBlk,
                            kOne = kA + kB + 512;
  __align__(1024) uint8_t m[kBuffers * kOne];
};

template <typename T, bool WIDE>
__device__ inline void gemm_ring(const edl_fp8_gemm& g, int block, int blocks,
                                 uint8_t* smem) {
  constexpr int FM = 2, FN = 4;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fA0 = (wave >> 1) * FM, wB = (wave & 1) * 64;
  const Spot s = spot_of<RingLds::BM, RingLds::BN>(g, block, blocks);
  Loads<RingLds::BM, RingLds::BN, 4> loads(g, s, wave, lane);
  constexpr int kLoads = Loads<RingLds::BM, RingLds::BN, 4>::kAll;
  static_assert(kLoads == 7, "the waits below");
  const uint32_t lds0 =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  auto stage = [&](uint32_t buf) {
    const uint32_t at = lds0 + buf * RingLds::kOne;
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      loads.one(at, at + RingLds::kA, at + RingLds::kA + RingLds::kB, q);
  };
  const int rr = ((lane & 15) >> 2) * 16 + (lane & 3), q4 = lane >> 4;
  const uint32_t lo = rr * kBlk + ((q4 ^ swz(rr)) << 4);
  const uint32_t hi = rr * kBlk + (((q4 + 4) ^ swz(rr)) << 4);
  typedef Hand<FM, FN, WIDE> H;
  H h;
  h.clear();
  const uint32_t rows = H::row_of(fA0) * kBlk;

  stage(0);
  if (s.steps > 1) stage(1);
  uint32_t buf = 0, ahead = 2;
  for (int t = 0; t < s.steps; ++t) {
    if (t + 1 < s.steps)
      asm volatile("s_waitcnt vmcnt(7) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 2 < s.steps) stage(ahead);
    const uint8_t* p = smem + buf * RingLds::kOne;
    H::read_scales(p + RingLds::kA + RingLds::kB + (lane & 15) * 4, fA0, wB,
                   h.sa, h.sb);
#pragma unroll
    for (int i = 0; i < FM; ++i) h.a[i] = H::read(p, rows + lo, rows + hi, i);
#pragma unroll
    for (int k = 0; k < FN; ++k)
      h.b[k] = H::read(p, RingLds::kA + wB * kBlk + lo,
                       RingLds::kA + wB * kBlk + hi, k);
    h.widen_b();
#pragma unroll
    for (int i = 0; i < FM; ++i) h.products(i);
    buf = buf == 2 ? 0 : buf + 1;
    ahead = ahead == 2 ? 0 : ahead + 1;
  }
  write_tile<T, FM, FN>(g, s, h, smem, wave, lane, fA0, wB, true);
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256, 2) void gemm_ring_kernel(edl_fp8_gemm g) {
  __shared__ RingLds lds;
  gemm_ring<T, WIDE>(g, blockIdx.x, gridDim.x, lds.m);
}
// a backward pass's products, of which none decides a sign
template <typename T0, typename T1>
__global__ __launch_bounds__(256, 2) void gemm_ring_pair_kernel(
    edl_fp8_gemm g0, edl_fp8_gemm g1, int blocks0) {
  __shared__ RingLds lds;
  if ((int)blockIdx.x < blocks0)
    gemm_ring<T0, is_f32<T0>>(g0, blockIdx.x, blocks0, lds.m);
  else
    gemm_ring<T1, is_f32<T1>>(g1, blockIdx.x - blocks0, gridDim.x - blocks0,
                              lds.m);
}

// the two products of a backward pass in one launch, each of 128 x 128
template <typename T0, typename T1>
__global__ __launch_bounds__(256, 2) void gemm_pair_kernel(edl_fp8_gemm g0,
                                                           edl_fp8_gemm g1,
                                                           int blocks0) {
  __shared__ GemmLds<128> lds;
  if ((int)blockIdx.x < blocks0)
    gemm_tile<2, 2, 4, 4, T0, is_f32<T0>>(g0, blockIdx.x, blocks0, lds.m);
  else
    gemm_tile<2, 2, 4, 4, T1, is_f32<T1>>(g1, blockIdx.x - blocks0,
                                          gridDim.x - blocks0, lds.m);
}

// joins a product's splits in order; a thread takes 16 neighbours of a row
template <typename T>
__device__ inline void gemm_join_as(const edl_fp8_gemm& g, int64_t block) {
  const int64_t each = g.part_ld / 16;
  const int64_t id = block * 256 + threadIdx.x;
  if (id >= g.M * each) return;
  const int64_t m = id / each, n = (id % each) * 16;
  float v[16], bias[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = 0.f;
  for (int s = 0; s < g.splits; ++s) {
    const float* p = g.part + ((int64_t)s * g.M + m) * g.part_ld + n;
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      f32x4 u = *reinterpret_cast<const f32x4*>(p + k);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[k + q] += u[q];
    }
  }
  load_bias16(g, n, bias);
  epilogue16<T>(g, m, n, v, bias);
}
__device__ inline void gemm_join(const edl_fp8_gemm& g, int64_t block) {
  if (g.c_type == EDL_T_F32)
    gemm_join_as<float>(g, block);
  else if (g.c_type == EDL_T_BF16)
    gemm_join_as<__bf16>(g, block);
  else
    gemm_join_as<_Float16>(g, block);
}

// what is left when a pass's products are done: the joins of up to two of
// them, and a bias's gradient; each takes the blocks that it needs
__global__ __launch_bounds__(256) void finish_kernel(edl_fp8_finish f) {
  int64_t b = blockIdx.x;
  if (b < f.join_blocks[0]) return gemm_join(f.g[0], b);
  b -= f.join_blocks[0];
  if (b < f.join_blocks[1]) return gemm_join(f.g[1], b);
  column_sums(f.sums, f.tiles, f.C, f.out, f.out_type,
              b - f.join_blocks[1]);
}

// ------------------------------- few rows ---------------------------------
// At most 16 rows of x, as served requests come: x is quantised in the
// registers of the wave that multiplies it and the weights go from memory
// straight to the matrix instruction, so that a layer is one launch. A
// workgroup takes 16 columns; its 16 waves share the blocks of 128 between
// them and join through LDS in order, with a block's loads ahead of its turn
// (16 x 4096 x 4096 9.2 us, 10.1 without). Bound by the read of the weights.
constexpr int kFewWaves = 16;

// 32 neighbours of a row as e4m3 bytes, and the scale's byte of the 128 that
// the four lanes of a row hold together
template <typename T>
__device__ inline i32x8 round32(const T* x, int64_t ld, int64_t M, int K,
                                int row, int64_t k0, bool wide, int* scale) {
  float v[32];
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 32; k += 8)
    load_row8<T>(x, ld, M, K, row, k0 + k, wide, v + k);
#pragma unroll
  for (int k = 0; k < 32; ++k) m = max(m, finite_abs(v[k]));
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  *scale = scale_byte(m);
  const float inv = inverse_of(*scale);
  i32x8 a;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    a[k] = pack4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3], inv);
  return a;
}

// The same for 16-bit inputs of 32 whole neighbours: the largest by packed
// 16-bit integers and two values a conversion, a fifth of the instructions.
// Every workgroup rounds all of x, so they are what 16 rows cost: 16 x 4096 x
// 4096 2.2 us more without this.
template <typename T>
struct Halves;
template <>
struct Halves<__bf16> {
  static constexpr uint16_t not_finite = 0x7f80;
  static __device__ inline float value(uint32_t bits) {
    return __uint_as_float(bits << 16);
  }
  static __device__ inline u16x2 pack(u16x2 old, uint32_t two, float s,
                                      bool hi) {
    const bf16x2 x = __builtin_bit_cast(bf16x2, two);
    const s16x2 o = __builtin_bit_cast(s16x2, old);
    return __builtin_bit_cast(
        u16x2, hi ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, x, s, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, x, s, false));
  }
};
template <>
struct Halves<_Float16> {
  static constexpr uint16_t not_finite = 0x7c00;
  static __device__ inline float value(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  }
  static __device__ inline u16x2 pack(u16x2 old, uint32_t two, float s,
                                      bool hi) {
    const f16x2 x = __builtin_bit_cast(f16x2, two);
    const s16x2 o = __builtin_bit_cast(s16x2, old);
    return __builtin_bit_cast(
        u16x2, hi ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, x, s, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, x, s, false));
  }
};
// false where a value of the wave's is not finite
template <typename T>
__device__ inline bool round32_fast(const u32x4* w, int* scale, i32x8* a) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const u16x2 t =
        __builtin_bit_cast(u16x2, w[k >> 2][k & 3] & 0x7fff7fffu);
    m = __builtin_elementwise_max(m, t);
  }
  uint32_t top = m[0] > m[1] ? m[0] : m[1];
  top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  if (__any(top >= Halves<T>::not_finite)) return false;
  *scale = scale_byte(__float_as_uint(Halves<T>::value(top)));
  const float s = scale_value(*scale, 0);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    u16x2 o = {0, 0};
    o = Halves<T>::pack(o, w[k >> 1][(k & 1) * 2], s, false);
    o = Halves<T>::pack(o, w[k >> 1][(k & 1) * 2 + 1], s, true);
    (*a)[k] = __builtin_bit_cast(int, o);
  }
  return true;
}

template <typename T>
__global__ __launch_bounds__(kFewWaves * 64) void few_rows_kernel(
    edl_fp8_gemm g, const T* __restrict__ x, int64_t x_ld, int K, bool wide) {
  __shared__ f32x4 s[kFewWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = lane & 15, q4 = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + row < g.N ? n0 + row : g.N - 1;
  const int kbs = (int)(g.ld / kBlk);
  const uint8_t* pb = g.b + n * g.ld + q4 * 32;
  const uint8_t* ps = g.sb + scale_slot(n);
  // what the end needs and what the next block does are fetched ahead
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  if (wave == 0 && g.bias) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n0 + q4 * 4 + q < g.N)
        bias[q] = load_any(g.bias, n0 + q4 * 4 + q, g.bias_type);
  }
  constexpr bool kHalf = sizeof(T) == 2;
  i32x8 b_next;
  int sb_next;
  u32x4 w_next[4] = {};
  auto fetch = [&](int kb) {
    b_next = *reinterpret_cast<const i32x8*>(pb + (int64_t)kb * kBlk);
    sb_next = ps[(int64_t)kb * g.b_rp];
    if (kHalf && wide && (kb + 1) * kBlk <= K) {  // the wave alike
      const T* p = x + (row < g.M ? row : 0) * x_ld + (int64_t)kb * kBlk +
                   q4 * 32;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w_next[k] = *reinterpret_cast<const u32x4*>(p + k * 8);
    }
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (wave < kbs) fetch(wave);
  for (int kb = wave; kb < kbs; kb += kFewWaves) {
    const i32x8 b = b_next;
    const int sb = sb_next;
    u32x4 w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = w_next[k];
    if (kb + kFewWaves < kbs) fetch(kb + kFewWaves);
    const int64_t k0 = (int64_t)kb * kBlk + q4 * 32;
    i32x8 a;
    int sa;
    bool done = false;
    if constexpr (kHalf) {
      if (wide && (kb + 1) * kBlk <= K) done = round32_fast<T>(w, &sa, &a);
    }
    if (!done) a = round32<T>(x, x_ld, g.M, K, row, k0, wide, &sa);
    if (!kHalf)  // the result is in 32 bits
      acc = mfma_wide(widen(b, scale_value(sb, 0)),
                      widen(a, scale_value(sa, 0)), acc);
    else
      acc = mfma<0, 0>(b, a, acc, sb, sa);
  }
  s[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
  // lane: row `row` of C, columns n0 + q4*4 + 0..3
  f32x4 t = s[0][lane];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) {
    f32x4 u = s[w][lane];
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] += u[q];
  }
  if (row >= g.M) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    int64_t c = n0 + q4 * 4 + q;
    if (c >= g.N) continue;
    store_any(g.c, row * g.N + c, activate(t[q] + bias[q], g.act), g.c_type);
  }
}

int64_t tiles_of(const edl_fp8_quant& a) {
  return ((a.R + kBlk - 1) / kBlk) * ((a.C + kBlk - 1) / kBlk);
}

constexpr int64_t kManyTiles = 1024;  // four a CU

template <typename T, int ROWS>
void launch_quantize_by(const edl_fp8_quant& a, hipStream_t st) {
  dim3 grid((unsigned)tiles_of(a)), block(2048 / ROWS);
  if (a.tile)
    quantize_kernel<T, ROWS, true, false><<<grid, block, 0, st>>>(a);
  else if (a.deriv)
    quantize_kernel<T, ROWS, false, true><<<grid, block, 0, st>>>(a);
  else
    quantize_kernel<T, ROWS, false, false><<<grid, block, 0, st>>>(a);
}
template <typename T>
void launch_quantize(const edl_fp8_quant& a, hipStream_t st) {
  if (tiles_of(a) >= kManyTiles)
    launch_quantize_by<T, 8>(a, st);
  else
    launch_quantize_by<T, 4>(a, st);
}

template <typename TX, int ROWS>
void launch_quantize_pair(const edl_fp8_quant& x, const edl_fp8_quant& w,
                          hipStream_t st) {
  const int n = (int)tiles_of(x);
  dim3 grid((unsigned)(n + tiles_of(w))), block(2048 / ROWS);
  if (w.type == EDL_T_F32)
    quantize_pair_kernel<TX, float, ROWS><<<grid, block, 0, st>>>(x, w, n);
  else if (w.type == EDL_T_BF16)
    quantize_pair_kernel<TX, __bf16, ROWS><<<grid, block, 0, st>>>(x, w, n);
  else
    quantize_pair_kernel<TX, _Float16, ROWS><<<grid, block, 0, st>>>(x, w, n);
}
template <int ROWS>
void launch_quantize_pair_by(const edl_fp8_quant& x, const edl_fp8_quant& w,
                             hipStream_t st) {
  if (x.type == EDL_T_F32)
    launch_quantize_pair<float, ROWS>(x, w, st);
  else if (x.type == EDL_T_BF16)
    launch_quantize_pair<__bf16, ROWS>(x, w, st);
  else
    launch_quantize_pair<_Float16, ROWS>(x, w, st);
}

int64_t tiles_of(const edl_fp8_gemm& g, int64_t bm, int64_t bn) {
  return ((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn);
}
int64_t tiles_of(const edl_fp8_gemm& g) {
  return g.tile == EDL_TILE_RING  ? tiles_of(g, 64, 128)
         : g.tile == EDL_TILE_128 ? tiles_of(g, 128, 128)
                                  : tiles_of(g, 256, 256);
}

}  // namespace

extern "C" int edl_fp8_quantize(const edl_fp8_quant* a, hipStream_t st) {
  if (a->type == EDL_T_F32)
    launch_quantize<float>(*a, st);
  else if (a->type == EDL_T_BF16)
    launch_quantize<__bf16>(*a, st);
  else
    launch_quantize<_Float16>(*a, st);
  return (int)hipGetLastError();
}

extern "C" int edl_fp8_quantize_pair(const edl_fp8_quant* x,
                                     const edl_fp8_quant* w, hipStream_t st) {
  if (tiles_of(*x) + tiles_of(*w) >= kManyTiles)
    launch_quantize_pair_by<8>(*x, *w, st);
  else
    launch_quantize_pair_by<4>(*x, *w, st);
  return (int)hipGetLastError();
}

// Chooses each product's tile, and how many splits of the contraction it
// takes, for n products (1 or 2, in one launch where their tiles agree).
//
// 256 x 256 reads each operand half as often but runs one workgroup a CU, so
// it takes the products that give each of the 256 CUs one. (In 32 bits a
// wave's fragments take twice the registers: no.) Where 128 x 128 leaves CUs
// without work, the ring of 64 x 128 is in time what its loads take: 4096 x
// 624 x 400 10.8 us in 128 tiles of 128, 7.6 in 256 of the ring, and in 32
// bits 14.0 and 9.9. Large products in 32 bits reach 1.18 PFLOP/s (16384 x
// 4096 x 4096 465 us, in 8 bits 240).
//
// Splits, up to 512 workgroups in all (two a CU): a join is a launch more,
// so a split has at least 8 blocks to do, or 4 where something else needs
// the launch that joins (finish).
extern "C" void edl_fp8_gemm_plan(edl_fp8_gemm* g, int n, int finish) {
  bool ring = true;
  for (int i = 0; i < n; ++i) {
    g[i].splits = 1;
    g[i].tile = !g[i].wide && tiles_of(g[i], 256, 256) >= 256
                    ? EDL_TILE_256
                    : EDL_TILE_128;
    if (g[i].tile == EDL_TILE_256 || tiles_of(g[i], 128, 128) >= 256)
      ring = false;
  }
  for (int i = 0; i < n; ++i)
    if (ring) g[i].tile = EDL_TILE_RING;
  for (int64_t least = finish ? 4 : 8; least < (1 << 20); least *= 2) {
    int64_t all = 0;
    for (int i = 0; i < n; ++i) {
      if (g[i].tile == EDL_TILE_256) continue;
      int64_t splits = g[i].ld / kBlk / least;
      splits = splits < 1 ? 1 : splits > 64 ? 64 : splits;
      g[i].splits = (int)splits;
      all += tiles_of(g[i]) * splits;
    }
    if (all <= 512) break;
  }
}

template <typename T, bool WIDE>
static void launch_as(const edl_fp8_gemm& g, hipStream_t st) {
  dim3 grid((unsigned)(tiles_of(g) * g.splits));
  if (g.tile == EDL_TILE_RING)
    gemm_ring_kernel<T, WIDE><<<grid, dim3(256), 0, st>>>(g);
  else if (g.tile == EDL_TILE_128)
    gemm_kernel<2, 2, 4, 4, T, WIDE><<<grid, dim3(256), 0, st>>>(g);
  else if constexpr (!WIDE)
    gemm_kernel<2, 4, 8, 4, T, false><<<grid, dim3(512), 0, st>>>(g);
}
template <typename T>
static void launch_half(const edl_fp8_gemm& g, hipStream_t st) {
  if (g.wide)
    launch_as<T, true>(g, st);
  else
    launch_as<T, false>(g, st);
}
static int launch_one(const edl_fp8_gemm& g, hipStream_t st) {
  if (g.c_type == EDL_T_F32)
    launch_as<float, true>(g, st);
  else if (g.c_type == EDL_T_BF16)
    launch_half<__bf16>(g, st);
  else
    launch_half<_Float16>(g, st);
  return (int)hipGetLastError();
}
template <typename T0, typename T1>
static void launch_pair(const edl_fp8_gemm* g, hipStream_t st) {
  const int b0 = (int)tiles_of(g[0]) * g[0].splits;
  const int b1 = (int)tiles_of(g[1]) * g[1].splits;
  dim3 grid((unsigned)(b0 + b1)), block(256);
  if (g[0].tile == EDL_TILE_RING)
    gemm_ring_pair_kernel<T0, T1><<<grid, block, 0, st>>>(g[0], g[1], b0);
  else
    gemm_pair_kernel<T0, T1><<<grid, block, 0, st>>>(g[0], g[1], b0);
}
template <typename T0>
static void launch_pair_as(const edl_fp8_gemm* g, hipStream_t st) {
  if (g[1].c_type == EDL_T_F32)
    launch_pair<T0, float>(g, st);
  else if (g[1].c_type == EDL_T_BF16)
    launch_pair<T0, __bf16>(g, st);
  else
    launch_pair<T0, _Float16>(g, st);
}

// n products (0 to 2), their joins, and where f's sums are not null a
// bias's gradient
extern "C" int edl_fp8_gemm_run(edl_fp8_finish* f, int n, hipStream_t st) {
  edl_fp8_gemm* g = f->g;
  int rc = 0;
  if (n == 2 && g[0].tile == g[1].tile && g[0].tile != EDL_TILE_256) {
    if (g[0].c_type == EDL_T_F32)
      launch_pair_as<float>(g, st);
    else if (g[0].c_type == EDL_T_BF16)
      launch_pair_as<__bf16>(g, st);
    else
      launch_pair_as<_Float16>(g, st);
    rc = (int)hipGetLastError();
  } else {
    for (int i = 0; i < n && rc == 0; ++i) rc = launch_one(g[i], st);
  }
  if (rc != 0) return rc;
  int64_t blocks = 0;
  for (int i = 0; i < 2; ++i) {
    f->join_blocks[i] =
        i < n && g[i].splits > 1
            ? (g[i].M * (g[i].part_ld / 16) + 255) / 256
            : 0;
    blocks += f->join_blocks[i];
  }
  if (f->sums) blocks += (f->C + 15) / 16;
  if (blocks == 0) return 0;
  finish_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(*f);
  return (int)hipGetLastError();
}

extern "C" int edl_fp8_few_rows(const edl_fp8_gemm* g, const void* x,
                                int64_t x_ld, int K, int x_type, int wide,
                                hipStream_t st) {
  dim3 grid((unsigned)((g->N + 15) / 16)), block(kFewWaves * 64);
  if (x_type == EDL_T_F32)
    few_rows_kernel<float><<<grid, block, 0, st>>>(
        *g, static_cast<const float*>(x), x_ld, K, wide);
  else if (x_type == EDL_T_BF16)
    few_rows_kernel<__bf16><<<grid, block, 0, st>>>(
        *g, static_cast<const __bf16*>(x), x_ld, K, wide);
  else
    few_rows_kernel<_Float16><<<grid, block, 0, st>>>(
        *g, static_cast<const _Float16*>(x), x_ld, K, wide);
  return (int)hipGetLastError();
}
