// Tiles of attention on MFMA 32x32x16: rows fetched into registers and stored to LDS,
// fragments read back by row or transposed, scores formed transposed (a lane holds 16 of
// one query), so that packing to bf16 makes them the next product's operand.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16v8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16v4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16v2;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((address_space(3))) bf16v4 lds_bf16v4;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int WROWS = 32;   // rows a wave owns

DEV_INLINE f32x16 mfma(bf16v8 a, bf16v8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

DEV_INLINE f32x16 zero16() {
  f32x16 z;
  #pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// maximum and sum over the two half-waves
DEV_INLINE float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
DEV_INLINE float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the wave's number as a scalar, so that branches on its rows are scalar too
DEV_INLINE int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <int D>
DEV_INLINE int swz(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3)
                  : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// One ROWS x D tile: fetched into registers, then stored to LDS.
template <int D, int ROWS, int NT>
struct Tile {
  static constexpr int UN = D / 8, STEP = NT / UN;     // rows NT threads cover
  static constexpr int PER = ROWS / STEP;
  static_assert(NT % UN == 0 && ROWS % STEP == 0, "tile does not divide");
  u32x4 r[PER];

  // base is wave-uniform: a full tile's loads share one lane offset. Rows past
  // the end repeat the last one, their weights are zero. (A branch around
  // each load would make the loads wait for one another.)
  DEV_INLINE void fetch(const __hip_bfloat16* base, int stride_t, int valid) {
    const int row = threadIdx.x / UN, cu = threadIdx.x % UN;
    if (valid >= ROWS) {
      const int off = row * stride_t + cu * 8;
      #pragma unroll
      for (int i = 0; i < PER; ++i)
        r[i] = *reinterpret_cast<const u32x4*>(base + (int64_t)(i * STEP) * stride_t + off);
    } else {
      #pragma unroll
      for (int i = 0; i < PER; ++i)
        r[i] = *reinterpret_cast<const u32x4*>(base + min(i * STEP + row, valid - 1) * stride_t
                                               + cu * 8);
    }
  }
  DEV_INLINE void store(char* lds) const {
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int row = i * STEP + threadIdx.x / UN, cu = threadIdx.x % UN;
      *reinterpret_cast<u32x4*>(lds + row * (2 * D) + ((cu ^ swz<D>(row)) << 4)) = r[i];
    }
  }
};

// A tile whose loads take one 32-bit offset a lane: rows past the end read as zero.
template <int D, int ROWS, int NT>
struct Rows : Tile<D, ROWS, NT> {
  using T = Tile<D, ROWS, NT>;
  int off;          // bytes, of this lane's first 16

  DEV_INLINE explicit Rows(int stride_t)
      : off(((int)threadIdx.x / T::UN * stride_t + (int)threadIdx.x % T::UN * 8) * 2) {}

  DEV_INLINE void fetch(const __hip_bfloat16* base, int stride_t, int valid) {
    // stride_t < 2^24: 64 rows stay within 2^31 bytes
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<__hip_bfloat16*>(base), 0, ((min(valid, ROWS) - 1) * stride_t + D) * 2, 0x00027000);
    #pragma unroll
    for (int i = 0; i < T::PER; ++i)
      this->r[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + i * T::STEP * stride_t * 2, 0, 0);
  }
};

// Lane offsets of the two kinds of fragment of a tile.
template <int D>
struct Frags {
  int row_off;         // row fragment: row l&31, chunk h
  int tr_lo, tr_hi;    // transpose reads: rows 4h + (l&15)/4 and 8 further

  DEV_INLINE Frags() {
    const int l = threadIdx.x & 63, h = l >> 5;
    const int row = l & 31;
    row_off = row * (2 * D) + ((h ^ swz<D>(row)) << 4);
    const int x = ((l >> 4) & 1) * 2 + ((l & 3) >> 1);
    const int r0 = 4 * h + ((l & 15) >> 2), r1 = r0 + 8;
    tr_lo = r0 * (2 * D) + ((x ^ swz<D>(r0)) << 4) + (l & 1) * 8;
    tr_hi = r1 * (2 * D) + ((x ^ swz<D>(r1)) << 4) + (l & 1) * 8;
  }
  // rows sub*32 + (l&31), elements ks*16 + h*8 ..
  DEV_INLINE bf16v8 row(const char* lds, int sub, int ks) const {
    return *reinterpret_cast<const bf16v8*>(lds + sub * (32 * 2 * D) + (row_off ^ (ks << 5)));
  }
  // element column dt*32 + (l&31), rows k0 + {4h.., 8+4h..}; k0 % 16 == 0
  DEV_INLINE bf16v8 col(char* lds, int k0, int dt) const {
    char* p = lds + k0 * (2 * D);
    const bf16v4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (lds_bf16v4*)(p + (tr_lo ^ (dt << 6))));
    const bf16v4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (lds_bf16v4*)(p + (tr_hi ^ (dt << 6))));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// two floats rounded to nearest even (v_cvt_pk_bf16_f32)
DEV_INLINE bf16v2 round2(float a, float b) {
  return __builtin_convertvector(f32x2{a, b}, bf16v2);
}

// accumulator rows 8*k .. 8*k+7 of this lane as bf16 k-slots of a 16-row step
DEV_INLINE bf16v8 pack8(const f32x16& s, int k) {
  bf16v8 out;
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bf16v2 v = round2(s[8 * k + 2 * j], s[8 * k + 2 * j + 1]);
    out[2 * j] = v[0];
    out[2 * j + 1] = v[1];
  }
  return out;
}

// row index within a 32-row block of accumulator register r
DEV_INLINE int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// this lane's row of a (rows, D) operand as fragments
template <int D>
DEV_INLINE void load_row(bf16v8 (&f)[D / 16], const __hip_bfloat16* base, int stride_t, int row) {
  const int h = (threadIdx.x & 63) >> 5;
  #pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    f[ks] = *reinterpret_cast<const bf16v8*>(base + (int64_t)row * stride_t + ks * 16 + h * 8);
}

// Waits for fragments here: left to their first use, in a loop, the wait would be
// for the loop's own loads as well, in every step.
template <int D>
DEV_INLINE void arrived(bf16v8 (&f)[D / 16]) {
  #pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    u32x4 x = __builtin_bit_cast(u32x4, f[ks]);
    asm volatile("" : "+v"(x));
    f[ks] = __builtin_bit_cast(bf16v8, x);
  }
}

// acc[dt] holds X^T (rows d, column = this lane's row): write the row times f.
// Two half-waves hold alternating groups of four d; one swap makes 16 B runs.
template <int D>
DEV_INLINE void store_rows(const f32x16 (&acc)[D / 32], float f, __hip_bfloat16* row, bool valid) {
  const int h = (threadIdx.x & 63) >> 5;
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    #pragma unroll
    for (int g = 0; g < 2; ++g) {       // d 16g .. 16g+15 of the 32
      uint32_t w[4];
      #pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = __builtin_bit_cast(
            uint32_t, round2(acc[dt][8 * g + 2 * j] * f, acc[dt][8 * g + 2 * j + 1] * f));
      }
      const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      if (valid)
        *reinterpret_cast<u32x4*>(row + dt * 32 + g * 16 + h * 8) = u32x4{x[0], y[0], x[1], y[1]};
    }
  }
}

// The same rows in fp32 (partial sums of a head split).
template <int D>
DEV_INLINE void store_rows_f32(const f32x16 (&acc)[D / 32], float* row, bool valid) {
  const int h = (threadIdx.x & 63) >> 5;
  if (!valid) return;
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
    #pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(row + dt * 32 + g * 8 + h * 4) =
          f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
}

}  // namespace
