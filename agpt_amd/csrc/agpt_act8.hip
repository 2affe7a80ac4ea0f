// agpt_act8.hip — 8-bit activation checkpoints (gfx950): packing, unpacking,
// and the weight gradient of a linear layer from its checkpointed input.
//
// Packing and unpacking are HBM-bound: a lane packs 16 bytes of eight rows (eight
// loads in flight), the lanes of 32 columns share their blocks' scales, and a
// lane's codes are 32 consecutive bytes (64 in bf16). Packing 2^20 rows of 512
// fp32 takes 519 us (2.7 GB at 5.2 TB/s), unpacking 300K 128 us (6.0 TB/s).
//
// The weight gradient dW[o][i] = sum_t dy[t][o] val[t][i] contracts over rows
// that are far apart in memory. A matrix instruction takes from each lane
// eight consecutive steps of the contraction for one row of its operand, so a
// lane simply loads eight rows of its own columns: no transposition, no LDS,
// and any assignment of columns to operand rows is as good as another, so
// lane l takes columns 2l, 2l+1 of dy and 4l..4l+3 of the checkpoint, whose
// bytes lie together in its layout. A wave owns a 64 x 128 tile of dW (eight
// 32x32 accumulators) over a chunk of rows and needs no other wave.
//   val has at most 8 significant bits: exact in bf16.
//   an fp32 dy is cut into three bf16 parts by truncation, 8 + 8 + 8 bits,
//   which add up to it exactly: three products at the bf16 rate instead of one
//   at the fp32 rate, 1/16 of it.
// Chunks leave partial tiles, folded in chunk order. Behind a ReLU (2^20 rows of
// 512, input 128) HBM bounds it: 969 us, 5.0 GB at 5.1 TB/s. The wider layers'
// form below is bound by the matrix units: 128 x 512 over 2^20 rows in 339-358 us,
// 412 GFLOP of bf16 products at 1.15-1.2 PFLOP/s, where a library product of 8192^3
// reaches 1.14; 1000 x 1024 over 64K rows of bf16 in 173-205 us, 0.66-0.78, with
// LDS traffic beside it (operands out of it at three quarters of its rate).

#include "rows.h"
#include "../../include/agpt_act8.h"

#include <type_traits>

namespace {

using namespace agpt_rows;

constexpr int kThreads = 256;
constexpr int kBlock = 32;  // columns under one scale
constexpr int kRows = 8;    // rows of a layout block

int64_t row_blocks(int64_t T) { return (T + kRows - 1) / kRows; }

// ---- pack -------------------------------------------------------------------
// The scale byte of a block whose largest magnitude has the bits `m`: with
// top = 127 = 1.984375 * 2^6 (255 = 1.9921875 * 2^7), the exponent of m less
// that of top, one more if m's mantissa is above top's. 255 for infinity, NaN and
// what would need s above 2^120, whose codes' values need not be finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t m, bool relu) {
  if (m >= 0x7f800000u) return 255u;
  const int e = static_cast<int>((m + (relu ? 0x0000ffffu : 0x0001ffffu)) >> 23) - (relu ? 7 : 6);
  return e > 247 ? 255u : static_cast<uint32_t>(e < 1 ? 1 : e);
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, false));
  return v > o ? v : o;
}

// The larger of m and the magnitude bits of x that count for the block's scale:
// |x|, or x where it is above zero; what is not finite always counts (`all`
// collects |x| for that).
template <bool kRelu>
__device__ __forceinline__ void magnitude(float x, uint32_t& m, uint32_t& all) {
  const uint32_t b = __float_as_uint(x), a = b & 0x7fffffffu;
  if constexpr (kRelu) {
    const int s = static_cast<int>(b) > static_cast<int>(m) ? static_cast<int>(b) : static_cast<int>(m);
    m = static_cast<uint32_t>(s);  // (negative numbers are negative integers; m starts at 0)
    all = all > a ? all : a;
  } else {
    m = m > a ? m : a;
  }
}

// Four codes as bytes. Adding x / s to 1.5 * 2^23 (+ 128) rounds it to an integer,
// ties to even, in the sum's low byte: one fused multiply-add, and x / s is exact.
template <bool kRelu>
__device__ __forceinline__ uint32_t codes_of(const float* v, float inv) {
  constexpr float kBase = kRelu ? 12582912.0f : 12582912.0f + 128.0f;
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[j] = __float_as_uint(fmaf(v[j], inv, kBase));
    if constexpr (kRelu) {  // at least 1 above zero, 0 elsewhere
      const int low = static_cast<int>(__float_as_uint(kBase)) + (v[j] > 0.0f ? 1 : 0);
      b[j] = static_cast<uint32_t>(static_cast<int>(b[j]) > low ? static_cast<int>(b[j]) : low);
    }
  }
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return lo | hi;
}
// The codes of a block that is not finite: only a ReLU's mask is kept.
template <bool kRelu>
__device__ __forceinline__ uint32_t codes_of_nan(const float* v) {
  if constexpr (!kRelu) return 0x80808080u;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = __float_as_uint(v[j]);
    if (!(b >> 31) && b != 0u && b <= 0x7f800000u) w |= 1u << (8 * j);
  }
  return w;
}

// A lane holds eight rows of V columns (V 1: of four, element by element).
template <typename T, int V, bool kRelu>
__global__ __launch_bounds__(kThreads) void pack_kernel(const T* __restrict__ x, int64_t ld, uint8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ scales, int64_t rows, int pieces,
                                                        int64_t items, int gx) {
  constexpr int kCols = V == 1 ? 4 : V, kQuads = kCols / 4, kLanes = kBlock / kCols;  // lanes that share a block
  for (int64_t i = static_cast<int64_t>(block_x()) * kThreads + thread_x(); i < items;
       i += static_cast<int64_t>(gx) * kThreads) {
    const int64_t rb = i / pieces;
    const int q = static_cast<int>(i - rb * pieces);
    const T* p = x + rb * kRows * ld + kCols * q;
    const int live = rows - rb * kRows < kRows ? static_cast<int>(rows - rb * kRows) : kRows;
    Raw<T, kCols> raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      raw[r].zero();
      if (r < live) {
        if constexpr (V > 1) {
          raw[r].load(p + r * ld);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[r].w[j] = __float_as_uint(p[r * ld + j]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j += 2)
            raw[r].w[j / 2] = p[r * ld + j].bits | static_cast<uint32_t>(p[r * ld + j + 1].bits) << 16;
        }
      }
    }
    uint32_t c[kQuads][kRows], sb[2] = {0u, 0u};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float v[kCols];
      raw[r].get(v);
      uint32_t m = 0, all = 0;
#pragma unroll
      for (int j = 0; j < kCols; ++j) magnitude<kRelu>(v[j], m, all);
      if (kRelu && all >= 0x7f800000u) m = all;
      m = dpp_max<0x1B>(dpp_max<0xB1>(m));
      if constexpr (kLanes == 8) m = dpp_max<0x141>(m);
      const uint32_t e = scale_byte(m, kRelu);
      const float inv = __uint_as_float((e == 255u ? 0u : 254u - e) << 23);  // 1 / s = 2^(127 - e)
#pragma unroll
      for (int k = 0; k < kQuads; ++k) c[k][r] = codes_of<kRelu>(v + 4 * k, inv);
      if (e == 255u) {
#pragma unroll
        for (int k = 0; k < kQuads; ++k) c[k][r] = codes_of_nan<kRelu>(v + 4 * k);
      }
      sb[r / 4] |= e << (8 * (r % 4));
    }
    uint4* out = reinterpret_cast<uint4*>(codes + i * (kCols * kRows));
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      out[2 * k] = uint4{c[k][0], c[k][1], c[k][2], c[k][3]};
      out[2 * k + 1] = uint4{c[k][4], c[k][5], c[k][6], c[k][7]};
    }
    if (q % kLanes == 0) *reinterpret_cast<uint2*>(scales + (i / kLanes) * kRows) = uint2{sb[0], sb[1]};
  }
}

// ---- values -------------------------------------------------------------------
// s = 2^(e - 127); e = 255 reads as infinity, and every value as NaN: code * inf - zero * inf.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
template <int kByte>
__device__ __forceinline__ float byte_f(uint32_t w) {
  return static_cast<float>((w >> (8 * kByte)) & 0xffu);
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void unpack_kernel(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, T* __restrict__ x,
                                                          int64_t ld, int64_t rows, int quads, int64_t items, int gx,
                                                          float zero) {
  for (int64_t i = static_cast<int64_t>(block_x()) * kThreads + thread_x(); i < items;
       i += static_cast<int64_t>(gx) * kThreads) {
    const int64_t rb = i / quads;
    const int q = static_cast<int>(i - rb * quads);
    const uint4 a = reinterpret_cast<const uint4*>(codes + i * (4 * kRows))[0];
    const uint4 b = reinterpret_cast<const uint4*>(codes + i * (4 * kRows))[1];
    const uint2 sc = *reinterpret_cast<const uint2*>(scales + (rb * (quads / 8) + q / 8) * kRows);
    const uint32_t c[kRows] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const int live = rows - rb * kRows < kRows ? static_cast<int>(rows - rb * kRows) : kRows;
    T* p = x + rb * kRows * ld + 4 * q;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float s = scale_of(((r < 4 ? sc.x : sc.y) >> (8 * (r % 4))) & 0xffu), z = -zero * s;
      const float v[4] = {fmaf(byte_f<0>(c[r]), s, z), fmaf(byte_f<1>(c[r]), s, z), fmaf(byte_f<2>(c[r]), s, z),
                          fmaf(byte_f<3>(c[r]), s, z)};
      if (r < live) {
        if constexpr (V == 4) {
          store_row<4>(p + r * ld, v);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float one[1] = {v[j]};
            store_row<1>(p + r * ld + j, one);
          }
        }
      }
    }
  }
}

// ---- weight gradient --------------------------------------------------------------
constexpr int kTileO = 64, kTileI = 128, kStep = 16;  // a wave's tile of dW, rows of a step

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The upper halves of two words as a pair of bf16, the first one low.
__device__ __forceinline__ uint32_t high_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t low_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }

struct Grad {
  int64_t rows, ld, chunk_rows;
  int out, in, tiles_o, tiles_i, chunks;
  float zero;
};

// What a lane holds of a step: its eight rows of two columns of dy, of four
// code columns with their scales, and of the ReLU's codes.
template <typename T>
struct Held {
  uint32_t a[kRows][sizeof(T) == 4 ? 2 : 1];
  uint4 c0, c1;
  uint2 sc;
  uint4 h0, h1;
};

// Two columns of a row in one load, at the alignment of one (which global loads
// do without): rows of an odd stride or base need no form of their own.
typedef uint32_t pair_f32 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t pair_bf16 __attribute__((aligned(2)));

// kPair: columns 2l and 2l + 1 in one load; otherwise (a width of 1)
// columns l and l + 32.
template <typename T, bool kPair, bool kRelu>
__global__ __launch_bounds__(kThreads, 2) void wgrad_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ hc,
                                                            T* __restrict__ dh, const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales,
                                                            float* __restrict__ dw, float* __restrict__ db,
                                                            int64_t db_ld, Grad g) {
  const int lane = thread_x() & 63, l = lane & 31, half = lane >> 5;
  // the wave's number is one for all its lanes: its rows' addresses are scalar,
  // and a lane adds one 32-bit offset that stays the same for every step
  const int wave = __builtin_amdgcn_readfirstlane(thread_x() >> 6);
  const int64_t unit = static_cast<int64_t>(block_x()) * (kThreads / 64) + wave;
  const int tiles = g.tiles_o * g.tiles_i;
  const int chunk = static_cast<int>(unit / tiles), tile = static_cast<int>(unit - static_cast<int64_t>(chunk) * tiles);
  if (chunk >= g.chunks) return;
  const int to = tile / g.tiles_i, ti = tile - to * g.tiles_i;
  const int o0 = to * kTileO, i0 = ti * kTileI;
  const int64_t t0 = chunk * g.chunk_rows, t1 = t0 + g.chunk_rows < g.rows ? t0 + g.chunk_rows : g.rows;
  const int oa = kPair ? o0 + 2 * l : o0 + l, ob = kPair ? oa + 1 : oa + 32;  // the lane's columns of dy
  const bool ina = oa < g.out, inb = ob < g.out;
  const int quads = g.in / 4, quad = i0 / 4 + l;
  const bool inq = quad < quads;
  const int64_t blocks = (g.rows + kRows - 1) / kRows;
  // A column past the edge is read as the last one: it only reaches entries of
  // dW, db and dh that are not written.
  // The last of an odd number of columns comes as the second of a pair.
  const bool second = kPair && oa == g.out - 1;
  const int ca = ina && !second ? oa : g.out - (kPair ? 2 : 1), cb = inb ? ob : g.out - 1, cq = inq ? quad : quads - 1;
  const uint32_t off_a = static_cast<uint32_t>(half * kRows * g.ld + ca) * sizeof(T);
  const uint32_t off_b = static_cast<uint32_t>(half * kRows * g.ld + cb) * sizeof(T);
  const uint32_t off_d = static_cast<uint32_t>(half * kRows * g.out + ca) * sizeof(T);
  const uint32_t off_c = static_cast<uint32_t>(half * quads + cq) * (4 * kRows);
  const uint32_t off_s = static_cast<uint32_t>(half * (quads / 8) + cq / 8) * kRows;
  const uint32_t off_h = static_cast<uint32_t>(half * (g.out / 4) + ca / 4) * (4 * kRows);

  f32x16 acc[2][4];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[p][j][r] = 0.0f;
  float sum_a = 0.0f, sum_b = 0.0f;
  const bool sums = db != nullptr && ti == 0, writes = kRelu && ti == 0;

  auto row = [&](const char* p, Held<T>& w, int r) {
    if constexpr (sizeof(T) == 4 && kPair) {
      const pair_f32 v = *reinterpret_cast<const pair_f32*>(p + off_a);
      w.a[r][0] = v.x;
      w.a[r][1] = v.y;
    } else if constexpr (sizeof(T) == 4) {
      w.a[r][0] = *reinterpret_cast<const uint32_t*>(p + off_a);
      w.a[r][1] = *reinterpret_cast<const uint32_t*>(p + off_b);
    } else if constexpr (kPair) {
      w.a[r][0] = *reinterpret_cast<const pair_bf16*>(p + off_a);
    } else {
      w.a[r][0] = *reinterpret_cast<const uint16_t*>(p + off_a) |
                  static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + off_b)) << 16;
    }
  };
  auto load = [&](int64_t t, Held<T>& w) {
    const char* p = reinterpret_cast<const char*>(dy + t * g.ld);
    const int64_t step = g.ld * static_cast<int64_t>(sizeof(T)), rb = t / kRows;
    const char* pc = reinterpret_cast<const char*>(codes) + rb * quads * (4 * kRows);
    const char* ps = reinterpret_cast<const char*>(scales) + rb * (quads / 8) * kRows;
    const char* ph = reinterpret_cast<const char*>(hc) + rb * (g.out / 4) * (4 * kRows);
    auto blocks_of = [&]() {
      w.c0 = *reinterpret_cast<const uint4*>(pc + off_c);
      w.c1 = *reinterpret_cast<const uint4*>(pc + off_c + 16);
      w.sc = *reinterpret_cast<const uint2*>(ps + off_s);
      if constexpr (kRelu) {
        w.h0 = *reinterpret_cast<const uint4*>(ph + off_h);
        w.h1 = *reinterpret_cast<const uint4*>(ph + off_h + 16);
      }
    };
    if (t + kStep <= t1) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) row(p + r * step, w, r);
      blocks_of();
      return;
    }
    // the last step of the last chunk: rows past the end are zeros, and so are the values of a block past it
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int c = 0; c < (sizeof(T) == 4 ? 2 : 1); ++c) w.a[r][c] = 0u;
      if (t + half * kRows + r < t1) row(p + r * step, w, r);
    }
    w.c0 = w.c1 = w.h0 = w.h1 = uint4{0u, 0u, 0u, 0u};
    w.sc = uint2{0u, 0u};
    if (rb + half < blocks) blocks_of();
  };

  auto step = [&](int64_t t, Held<T>& w) {
    if constexpr (kPair && !kRelu) {
      if (g.out & 1) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          w.a[r][0] = !second ? w.a[r][0] : (sizeof(T) == 4 ? w.a[r][sizeof(T) == 4 ? 1 : 0] : w.a[r][0] >> 16);
      }
    }
    if constexpr (kRelu) {
      const uint32_t h[kRows] = {w.h0.x, w.h0.y, w.h0.z, w.h0.w, w.h1.x, w.h1.y, w.h1.z, w.h1.w};
      const int sh = (l & 1) * 16;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const uint32_t m = h[r] >> sh;
        if constexpr (sizeof(T) == 4) {
          w.a[r][0] = (m & 0xffu) ? w.a[r][0] : 0u;
          w.a[r][1] = (m & 0xff00u) ? w.a[r][1] : 0u;
        } else {
          w.a[r][0] &= ((m & 0xffu) ? 0xffffu : 0u) | ((m & 0xff00u) ? 0xffff0000u : 0u);
        }
      }
      if (writes) {
        char* p = reinterpret_cast<char*>(dh + t * g.out);
        const int64_t drow = g.out * static_cast<int64_t>(sizeof(T));
        const bool whole = t + kStep <= t1;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          if (ina && (whole || t + half * kRows + r < t1)) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint2*>(p + r * drow + off_d) = uint2{w.a[r][0], w.a[r][1]};
            else *reinterpret_cast<uint32_t*>(p + r * drow + off_d) = w.a[r][0];
          }
        }
      }
    }
    if (sums) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if constexpr (sizeof(T) == 4) {
          sum_a += __uint_as_float(w.a[r][0]);
          sum_b += __uint_as_float(w.a[r][1]);
        } else {
          sum_a += __uint_as_float(w.a[r][0] << 16);
          sum_b += __uint_as_float(w.a[r][0] & 0xffff0000u);
        }
      }
    }
    // the four code columns as bf16, eight rows each
    uint4 b[4];
    {
      const uint32_t c[kRows] = {w.c0.x, w.c0.y, w.c0.z, w.c0.w, w.c1.x, w.c1.y, w.c1.z, w.c1.w};
      uint32_t v[4][kRows / 2];
#pragma unroll
      for (int r = 0; r < kRows; r += 2) {
        const uint32_t sw = r < 4 ? w.sc.x : w.sc.y;
        const float s0 = scale_of((sw >> (8 * (r % 4))) & 0xffu), z0 = -g.zero * s0;
        const float s1 = scale_of((sw >> (8 * (r % 4 + 1))) & 0xffu), z1 = -g.zero * s1;
        auto pair = [&](float x, float y) {
          return high_pair(__float_as_uint(fmaf(x, s0, z0)), __float_as_uint(fmaf(y, s1, z1)));
        };
        v[0][r / 2] = pair(byte_f<0>(c[r]), byte_f<0>(c[r + 1]));
        v[1][r / 2] = pair(byte_f<1>(c[r]), byte_f<1>(c[r + 1]));
        v[2][r / 2] = pair(byte_f<2>(c[r]), byte_f<2>(c[r + 1]));
        v[3][r / 2] = pair(byte_f<3>(c[r]), byte_f<3>(c[r + 1]));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = uint4{v[j][0], v[j][1], v[j][2], v[j][3]};
    }
    auto products = [&](int p, uint4 a) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[p][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b[j]),
                                                            acc[p][j], 0, 0, 0);
    };
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t m[kRows / 2];
      if constexpr (sizeof(T) == 4) {
        // three parts by truncation; each remainder is exact
        float x[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) x[r] = __uint_as_float(w.a[r][p]);
#pragma unroll
        for (int part = 0; part < 3; ++part) {
#pragma unroll
          for (int r = 0; r < kRows; r += 2) m[r / 2] = high_pair(__float_as_uint(x[r]), __float_as_uint(x[r + 1]));
          if (part < 2) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) x[r] -= __uint_as_float(__float_as_uint(x[r]) & 0xffff0000u);
          }
          products(p, uint4{m[0], m[1], m[2], m[3]});
        }
      } else {
#pragma unroll
        for (int r = 0; r < kRows; r += 2)
          m[r / 2] = p ? high_pair(w.a[r][0], w.a[r + 1][0]) : low_pair(w.a[r][0], w.a[r + 1][0]);
        products(p, uint4{m[0], m[1], m[2], m[3]});
      }
    }
  };

  Held<T> w0, w1;
  load(t0, w0);
  for (int64_t t = t0; t < t1; t += 2 * kStep) {
    if (t + kStep < t1) load(t + kStep, w1);
    step(t, w0);
    if (t + kStep < t1) {
      if (t + 2 * kStep < t1) load(t + 2 * kStep, w0);
      step(t + kStep, w1);
    }
  }

  // accumulator register r of lane (l, half): operand row 8 (r / 4) + 4 half + r % 4 of dy, column l of the codes
  float* out = dw + static_cast<int64_t>(chunk) * g.out * g.in;
  if (inq) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = 8 * (r / 4) + 4 * half + r % 4;
        const int o = kPair ? o0 + 2 * m + p : o0 + m + 32 * p;
        if (o < g.out)
          *reinterpret_cast<float4*>(out + static_cast<int64_t>(o) * g.in + 4 * quad) =
              float4{acc[p][0][r], acc[p][1][r], acc[p][2][r], acc[p][3][r]};
      }
  }
  if (sums) {
    sum_a += __shfl_xor(sum_a, 32);
    sum_b += __shfl_xor(sum_b, 32);
    if (half == 0) {
      if (ina) db[chunk * db_ld + oa] = sum_a;
      if (inb) db[chunk * db_ld + ob] = sum_b;
    }
  }
}

// ---- weight gradient, operands shared through LDS ------------------------------------
// Where dW is wider than a wave's tile, every wave of the kernel above cuts and
// decodes the same columns again. Here a workgroup of eight waves owns a
// (64 WO) x (128 WI) tile of dW, WO * WI = 8: per step of 32 rows each wave
// prepares a share of the operands once, in the lane layout of the matrix
// instruction, and puts them into LDS; then each wave multiplies its 64 x 128
// tile out of it. Two LDS buffers: step n is multiplied while step n + 1 is
// prepared and the rows of step n + 2 are on their way.
// An operand group is 64 columns: [octet of rows][part][column parity][32 lanes] of 16 bytes
// (eight rows of a column as bf16), written and read without bank conflicts.
constexpr int kShared = 512, kSRows = 32, kOctets = kSRows / kRows;

template <typename T, int WO, bool kRelu>
__global__ __launch_bounds__(kShared, 2) void wgrad_shared_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ hc,
                                                                  T* __restrict__ dh, const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales,
                                                                  float* __restrict__ dw, float* __restrict__ db,
                                                                  int64_t db_ld, Grad g, int grid) {
  constexpr int WI = 8 / WO, kParts = sizeof(T) == 4 ? 3 : 1;
  constexpr int kGroupA = kOctets * kParts * 2 * 32, kGroupB = kOctets * 2 * 32;  // uint4 each
  // A wave's jobs of eight rows: of dy with two columns a lane (kPair) or, where that would leave waves without, one;
  // of the codes with two.
  constexpr bool kPair = WO == 4;
  constexpr int kCols = kPair ? 2 : 1, kJobsA = WO / (2 * kCols), kJobsB = WI / 2;
  __shared__ uint4 sa[2][WO * kGroupA];
  __shared__ uint4 sb[2][2 * WI * kGroupB];
  const int lane = thread_x() & 63, l = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(thread_x() >> 6);
  const int tiles = g.tiles_o * g.tiles_i;
  // workgroups of one chunk on one XCD (they are dealt over eight in turn), whose L2 then holds the chunk's rows for all of them
  const int unit = (block_x() & 7) * (grid >> 3) + (block_x() >> 3);
  const int chunk = unit / tiles, tile = unit - chunk * tiles;
  if (chunk >= g.chunks) return;
  const int to = tile / g.tiles_i, ti = tile - to * g.tiles_i;
  const int o0 = to * 64 * WO, i0 = ti * 128 * WI;
  const int64_t t0 = chunk * g.chunk_rows, t1 = t0 + g.chunk_rows < g.rows ? t0 + g.chunk_rows : g.rows;
  const int quads = g.in / 4;
  const int64_t blocks = (g.rows + kRows - 1) / kRows;

  // This wave's share of the preparation. A column past the edge is read as the
  // last one: it only reaches entries of dW, db and dh that are not written.
  // The last of an odd number comes as the second of a pair.
  int ga[kJobsA], octa[kJobsA], cola[kJobsA];
  uint32_t off_a[kJobsA], off_d[kJobsA], off_h[kJobsA];
#pragma unroll
  for (int q = 0; q < kJobsA; ++q) {
    const int job = wave * kJobsA + q;
    ga[q] = kPair ? job >> 1 : job >> 2;
    octa[q] = kPair ? 2 * (job & 1) + half : job & 3;
    cola[q] = o0 + 64 * ga[q] + (kPair ? 2 * l : lane);
    const int c = cola[q] + kCols <= g.out ? cola[q] : g.out - kCols;
    off_a[q] = static_cast<uint32_t>(octa[q] * kRows * g.ld + c) * sizeof(T);
    off_d[q] = static_cast<uint32_t>(octa[q] * kRows * g.out + c) * sizeof(T);
    off_h[q] = static_cast<uint32_t>(octa[q] * (g.out / 4) + c / 4) * (4 * kRows);
  }
  int gb[kJobsB], octb[kJobsB];
  uint32_t off_c[kJobsB], off_s[kJobsB];
#pragma unroll
  for (int q = 0; q < kJobsB; ++q) {
    gb[q] = kJobsB == 1 ? wave >> 1 : wave;
    octb[q] = 2 * (kJobsB == 1 ? wave & 1 : q) + half;
    int quad = (i0 + 64 * gb[q]) / 4 + l / 2;
    quad = quad < quads ? quad : quads - 1;
    off_c[q] = static_cast<uint32_t>(octb[q] * quads + quad) * (4 * kRows);
    off_s[q] = static_cast<uint32_t>(octb[q] * (quads / 8) + quad / 8) * kRows;
  }
  const bool sums = db != nullptr && ti == 0, writes = kRelu && ti == 0;
  float sum[kJobsA][kCols];
#pragma unroll
  for (int q = 0; q < kJobsA; ++q)
#pragma unroll
    for (int c = 0; c < kCols; ++c) sum[q][c] = 0.0f;

  struct Held {
    uint32_t a[kJobsA][kRows][sizeof(T) == 4 ? kCols : 1];
    uint4 h[kJobsA][2], c[kJobsB][2];
    uint2 s[kJobsB];
  };
  auto load = [&](int64_t t, Held& w) {
    const int64_t rb = t / kRows, step = g.ld * static_cast<int64_t>(sizeof(T));
    const char* pa = reinterpret_cast<const char*>(dy + t * g.ld);
    const char* pc = reinterpret_cast<const char*>(codes) + rb * quads * (4 * kRows);
    const char* ps = reinterpret_cast<const char*>(scales) + rb * (quads / 8) * kRows;
    const char* ph = reinterpret_cast<const char*>(hc) + rb * (g.out / 4) * (4 * kRows);
    auto row = [&](int q, int r) {
      const char* p = pa + r * step + off_a[q];
      if constexpr (sizeof(T) == 4 && kPair) {
        const pair_f32 v = *reinterpret_cast<const pair_f32*>(p);
        w.a[q][r][0] = v.x;
        w.a[q][r][1] = v.y;
      } else if constexpr (sizeof(T) == 4) {
        w.a[q][r][0] = *reinterpret_cast<const uint32_t*>(p);
      } else if constexpr (kPair) {
        w.a[q][r][0] = *reinterpret_cast<const pair_bf16*>(p);
      } else {
        w.a[q][r][0] = *reinterpret_cast<const uint16_t*>(p);
      }
    };
    auto block_h = [&](int q) {
      w.h[q][0] = *reinterpret_cast<const uint4*>(ph + off_h[q]);
      w.h[q][1] = *reinterpret_cast<const uint4*>(ph + off_h[q] + 16);
    };
    auto block_c = [&](int q) {
      w.c[q][0] = *reinterpret_cast<const uint4*>(pc + off_c[q]);
      w.c[q][1] = *reinterpret_cast<const uint4*>(pc + off_c[q] + 16);
      w.s[q] = *reinterpret_cast<const uint2*>(ps + off_s[q]);
    };
    if (t + kSRows <= t1) {
#pragma unroll
      for (int q = 0; q < kJobsA; ++q) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) row(q, r);
        if constexpr (kRelu) block_h(q);
      }
#pragma unroll
      for (int q = 0; q < kJobsB; ++q) block_c(q);
      return;
    }
    // the last step of the last chunk: rows past the end are zeros, and so are the values of blocks past it
#pragma unroll
    for (int q = 0; q < kJobsA; ++q) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int c = 0; c < (sizeof(T) == 4 ? kCols : 1); ++c) w.a[q][r][c] = 0u;
        if (t + octa[q] * kRows + r < t1) row(q, r);
      }
      if constexpr (kRelu) {
        w.h[q][0] = w.h[q][1] = uint4{0u, 0u, 0u, 0u};
        if (rb + octa[q] < blocks) block_h(q);
      }
    }
#pragma unroll
    for (int q = 0; q < kJobsB; ++q) {
      w.c[q][0] = w.c[q][1] = uint4{0u, 0u, 0u, 0u};
      w.s[q] = uint2{0u, 0u};
      if (rb + octb[q] < blocks) block_c(q);
    }
  };

  auto put_a = [&](int64_t t, Held& w, int q, uint4* to_lds) {
    auto& ra = w.a[q];
    if constexpr (kPair && !kRelu) {
      const bool second = cola[q] == g.out - 1;
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        ra[r][0] = !second ? ra[r][0] : (sizeof(T) == 4 ? ra[r][sizeof(T) == 4 ? 1 : 0] : ra[r][0] >> 16);
    }
    if constexpr (kRelu) {
      const uint32_t h[kRows] = {w.h[q][0].x, w.h[q][0].y, w.h[q][0].z, w.h[q][0].w,
                                 w.h[q][1].x, w.h[q][1].y, w.h[q][1].z, w.h[q][1].w};
      const int sh = kPair ? (l & 1) * 16 : (lane & 3) * 8;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const uint32_t m = h[r] >> sh;
        if constexpr (sizeof(T) == 4 || !kPair) {
          ra[r][0] = (m & 0xffu) ? ra[r][0] : 0u;
          if constexpr (kPair) ra[r][1] = (m & 0xff00u) ? ra[r][1] : 0u;
        } else {
          ra[r][0] &= ((m & 0xffu) ? 0xffffu : 0u) | ((m & 0xff00u) ? 0xffff0000u : 0u);
        }
      }
      if (writes) {
        char* p = reinterpret_cast<char*>(dh + t * g.out);
        const int64_t drow = g.out * static_cast<int64_t>(sizeof(T));
        const bool whole = t + kSRows <= t1;
        if (cola[q] < g.out) {
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if (whole || t + octa[q] * kRows + r < t1) {
              char* d = p + r * drow + off_d[q];
              if constexpr (sizeof(T) == 4 && kPair) *reinterpret_cast<uint2*>(d) = uint2{ra[r][0], ra[r][1]};
              else if constexpr (sizeof(T) == 4 || kPair) *reinterpret_cast<uint32_t*>(d) = ra[r][0];
              else *reinterpret_cast<uint16_t*>(d) = static_cast<uint16_t>(ra[r][0]);
            }
          }
        }
      }
    }
    if (sums) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) sum[q][c] += __uint_as_float(ra[r][c]);
        } else {
          sum[q][0] += __uint_as_float(ra[r][0] << 16);
          if constexpr (kPair) sum[q][1] += __uint_as_float(ra[r][0] & 0xffff0000u);
        }
      }
    }
    uint4* out = to_lds + ga[q] * kGroupA + octa[q] * (kParts * 64) + l;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int p = kPair ? c : half;
      uint32_t m[kRows / 2];
      if constexpr (sizeof(T) == 4) {
        float x[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) x[r] = __uint_as_float(ra[r][c]);
#pragma unroll
        for (int part = 0; part < 3; ++part) {
#pragma unroll
          for (int r = 0; r < kRows; r += 2) m[r / 2] = high_pair(__float_as_uint(x[r]), __float_as_uint(x[r + 1]));
          if (part < 2) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) x[r] -= __uint_as_float(__float_as_uint(x[r]) & 0xffff0000u);
          }
          out[(part * 2 + p) * 32] = uint4{m[0], m[1], m[2], m[3]};
        }
      } else {
#pragma unroll
        for (int r = 0; r < kRows; r += 2)
          m[r / 2] = c ? high_pair(ra[r][0], ra[r + 1][0]) : low_pair(ra[r][0], ra[r + 1][0]);
        out[p * 32] = uint4{m[0], m[1], m[2], m[3]};
      }
    }
  };
  auto put_b = [&](const Held& w, int q, uint4* to_lds) {
    const int sh = (l & 1) * 16;
    const uint32_t c[kRows] = {w.c[q][0].x >> sh, w.c[q][0].y >> sh, w.c[q][0].z >> sh, w.c[q][0].w >> sh,
                               w.c[q][1].x >> sh, w.c[q][1].y >> sh, w.c[q][1].z >> sh, w.c[q][1].w >> sh};
    uint32_t v[2][kRows / 2];
#pragma unroll
    for (int r = 0; r < kRows; r += 2) {
      const uint32_t sw = r < 4 ? w.s[q].x : w.s[q].y;
      const float s0 = scale_of((sw >> (8 * (r % 4))) & 0xffu), z0 = -g.zero * s0;
      const float s1 = scale_of((sw >> (8 * (r % 4 + 1))) & 0xffu), z1 = -g.zero * s1;
      v[0][r / 2] = high_pair(__float_as_uint(fmaf(byte_f<0>(c[r]), s0, z0)), __float_as_uint(fmaf(byte_f<0>(c[r + 1]), s1, z1)));
      v[1][r / 2] = high_pair(__float_as_uint(fmaf(byte_f<1>(c[r]), s0, z0)), __float_as_uint(fmaf(byte_f<1>(c[r + 1]), s1, z1)));
    }
    uint4* out = to_lds + gb[q] * kGroupB + octb[q] * 64 + l;
    out[0] = uint4{v[0][0], v[0][1], v[0][2], v[0][3]};
    out[32] = uint4{v[1][0], v[1][1], v[1][2], v[1][3]};
  };

  const int wo = wave / WI, wi = wave - wo * WI;
  f32x16 acc[2][4];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[p][j][r] = 0.0f;
  auto multiply = [&](const uint4* a, const uint4* b) {
    __builtin_amdgcn_s_setprio(2);  // over the preparation of the wave that shares the SIMD
    a += wo * kGroupA + l;
    b += 2 * wi * kGroupB + l;
#pragma unroll
    for (int ks = 0; ks < kOctets / 2; ++ks) {
      const int oct = 2 * ks + half;
      uint4 fb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) fb[j] = b[(j >> 1) * kGroupB + oct * 64 + (j & 1) * 32];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const uint4 fa = a[oct * (kParts * 64) + (part * 2 + p) * 32];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[p][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fa),
                                                                __builtin_bit_cast(bf16x8, fb[j]), acc[p][j], 0, 0, 0);
        }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto prepare = [&](int64_t t, Held& w, int buf) {
#pragma unroll
    for (int q = 0; q < kJobsA; ++q) put_a(t, w, q, sa[buf]);
#pragma unroll
    for (int q = 0; q < kJobsB; ++q) put_b(w, q, sb[buf]);
  };

  // Step n is multiplied from buffer n & 1 while step n + 1 is prepared and the
  // rows of the next kAhead steps are on their way: two where the registers hold
  // them (64K rows of 1024 x 1000 bf16 208 -> 179 us for one to two), one behind
  // a ReLU.
  constexpr int kAhead = kRelu ? 1 : 2;
  const int steps = static_cast<int>((t1 - t0 + kSRows - 1) / kSRows);
  auto at = [&](int n) { return t0 + static_cast<int64_t>(n) * kSRows; };
  Held w0, w1;
  if (steps > 0) load(at(0), w0);
  if (kAhead == 2 && steps > 1) load(at(1), w1);
  if (steps > 0) prepare(at(0), w0, 0);
  if (steps > kAhead) load(at(kAhead), w0);
  __syncthreads();
  int n = 0;
  if constexpr (kAhead == 1) {
    for (; n < steps; ++n) {
      const int buf = n & 1;
      multiply(sa[buf], sb[buf]);
      if (n + 1 < steps) prepare(at(n + 1), w0, buf ^ 1);
      if (n + 2 < steps) load(at(n + 2), w0);
      __syncthreads();
    }
  } else {
    auto body = [&](Held& w, int buf) {
      multiply(sa[buf], sb[buf]);
      prepare(at(n + 1), w, buf ^ 1);
      if (n + 3 < steps) load(at(n + 3), w);
      __syncthreads();
    };
    while (n + 1 < steps) {
      body(w1, 0);
      if (++n + 1 >= steps) break;
      body(w0, 1);
      ++n;
    }
    if (steps > 0) multiply(sa[n & 1], sb[n & 1]);
    __syncthreads();
  }

  float* out = dw + static_cast<int64_t>(chunk) * g.out * g.in;
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {
    const int i = i0 + 128 * wi + 64 * jj + 2 * l;
    if (i < g.in) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = 8 * (r / 4) + 4 * half + r % 4;
          const int o = o0 + 64 * wo + (kPair ? 2 * m + p : 32 * p + m);
          if (o < g.out)
            *reinterpret_cast<float2*>(out + static_cast<int64_t>(o) * g.in + i) =
                float2{acc[p][2 * jj][r], acc[p][2 * jj + 1][r]};
        }
    }
  }
  // db: a column's four octets of rows, added in order (the operands in LDS are no longer needed)
  if (sums) {
    float* s = reinterpret_cast<float*>(sa);
#pragma unroll
    for (int q = 0; q < kJobsA; ++q)
#pragma unroll
      for (int c = 0; c < kCols; ++c) s[octa[q] * (64 * WO) + cola[q] - o0 + c] = sum[q][c];
    __syncthreads();
    const int c = thread_x();
    if (c < 64 * WO && o0 + c < g.out) {
      float a = s[c];
      for (int q = 1; q < kOctets; ++q) a += s[q * (64 * WO) + c];
      db[chunk * db_ld + o0 + c] = a;
    }
  }
}

__global__ __launch_bounds__(kFoldThreads) void wgrad_fold_kernel(const float* __restrict__ part, int64_t n,
                                                                  const float* __restrict__ part_b, int64_t ldb,
                                                                  int chunks, int out, float* __restrict__ dw,
                                                                  float* __restrict__ db, int wblocks) {
  const int blk = block_x();
  if (blk < wblocks) {
    fold_columns(part + static_cast<int64_t>(blk) * 64, n, chunks,
                 n - static_cast<int64_t>(blk) * 64 < 64 ? static_cast<int>(n - static_cast<int64_t>(blk) * 64) : 64, 0,
                 dw + static_cast<int64_t>(blk) * 64);
  } else {
    fold_columns(part_b, ldb, chunks, out, blk - wblocks, db);
  }
}

// The fold of a large dW over few chunks: a thread per four columns, all chunks'
// loads in flight, and db by the last workgroups.
__global__ __launch_bounds__(kThreads) void wgrad_add_kernel(const float* __restrict__ part, int64_t n,
                                                             const float* __restrict__ part_b, int64_t ldb, int chunks,
                                                             int out, float* __restrict__ dw, float* __restrict__ db,
                                                             int wblocks) {
  const int blk = block_x();
  if (blk < wblocks) {
    const int64_t c = (static_cast<int64_t>(blk) * kThreads + thread_x()) * 4;
    if (c >= n) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
    for (int q = 0; q < chunks; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(part + q * n + c);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    *reinterpret_cast<float4*>(dw + c) = a;
  } else {
    const int c = (blk - wblocks) * kThreads + thread_x();
    if (c >= out) return;
    float a = 0.0f;
#pragma unroll 16
    for (int q = 0; q < chunks; ++q) a += part_b[q * ldb + c];
    db[c] = a;
  }
}

constexpr int kUnits = 2048;      // waves: two per SIMD
constexpr int kMinRows = 64;      // of a chunk
// Where a thread per four columns folds the chunks: enough threads to fill the
// chip, few enough loads each (1024 x 1000 over 16 chunks: 41 us by slots of rows,
// of which 48 of 64 idle, 11 so).
constexpr int64_t kAddWidth = int64_t{1} << 18;
constexpr int kAddChunks = 64;
constexpr int kOneChunk = 256;    // rows that one chunk takes: the fold's launch costs as much as the steps it saves
constexpr int kMaxWidth = 32768;

struct Plan {
  int wo;  // 0: a wave for itself; 2, 4: waves down the shared tile
  int tiles_o, tiles_i, chunks;
  int64_t chunk_rows, db_ld;
};
// Shared operands where dW is wider than a wave's tile in both directions and
// fills enough of the shared tile: one of those costs what kSharedTile of a wave's
// do (2^18 fp32 rows: 95 us a tile against 15.5). Measured on both sides of it, fp32
// and bf16 us, a wave alone | shared: 384 from 384 columns 285, 174 | 368, 183 (18
// tiles | 4: alone); 128 from 256 77, 50 | 95, 61 (4 | 1: alone); 129 from 256 96, 66
// | 99, 57 (6 | 1: shared); 200 from 256 132, 75 | 110, 65 (8 | 1: shared).
constexpr int kSharedTile = 6;
int shared_wo(int out, int in) {
  if (out <= kTileO || in <= kTileI) return 0;
  const int wo = out <= 2 * kTileO ? 2 : 4, to = kTileO * wo, ti = kTileI * (8 / wo);
  const int alone = ((out + kTileO - 1) / kTileO) * ((in + kTileI - 1) / kTileI);
  const int tiles = ((out + to - 1) / to) * ((in + ti - 1) / ti);
  return alone < kSharedTile * tiles ? 0 : wo;
}
Plan plan_of(int64_t T, int out, int in, int wo) {
  Plan p;
  p.wo = wo;
  const int to = wo ? 64 * wo : kTileO, ti = wo ? 128 * (8 / wo) : kTileI, step = wo ? kSRows : kStep;
  p.tiles_o = (out + to - 1) / to;
  p.tiles_i = (in + ti - 1) / ti;
  const int64_t tiles = static_cast<int64_t>(p.tiles_o) * p.tiles_i;
  int64_t chunks = (wo ? kUnits / 8 : kUnits) / tiles;
  if (chunks > (T + kMinRows - 1) / kMinRows) chunks = (T + kMinRows - 1) / kMinRows;
  if (chunks < 1 || T <= kOneChunk) chunks = 1;
  p.chunk_rows = ((T + chunks - 1) / chunks + step - 1) / step * step;
  if (p.chunk_rows < step) p.chunk_rows = step;
  p.chunks = static_cast<int>((T + p.chunk_rows - 1) / p.chunk_rows);
  if (p.chunks < 1) p.chunks = 1;
  p.db_ld = (out + 3) / 4 * 4;
  return p;
}

int check(const char* what, int64_t T, int64_t ld, int width, int W, int dtype) {
  if (T < 0 || width < 1) return invalid(what, "T < 0 or a width below 1");
  if (W < kBlock || W % kBlock != 0) return invalid(what, "a checkpoint's width must be a multiple of 32");
  if (W > kMaxWidth || width > kMaxWidth) {
    return agpt_internal_set_error(AGPT_ERR_UNSUPPORTED, "agpt_act8: widths above 32768 are not supported");
  }
  if (ld < width) return invalid(what, "row stride smaller than a row");
  if (dtype != AGPT_DTYPE_F32 && dtype != AGPT_DTYPE_BF16) return invalid(what, "unknown dtype");
  return AGPT_OK;
}

int grid_of(int64_t items) {
  const int64_t need = (items + kThreads - 1) / kThreads;
  return static_cast<int>(need < 4096 ? need : 4096);
}

int wgrad(const char* what, const void* dy, int64_t ld, int dtype, const uint8_t* hc, void* dh, const uint8_t* codes,
          const uint8_t* scales, int relu, float* dw, float* db, float* ws, int64_t ws_floats, int64_t T, int out, int in,
          void* stream) {
  if (const int rc = check(what, T, ld, out, in, dtype)) return rc;
  if (!dw || !ws || (T > 0 && (!dy || !codes || !scales))) return invalid(what, "null pointer");
  if (ws_floats < agpt_act8_wgrad_workspace_floats(T, out, in))
    return invalid(what, "workspace smaller than agpt_act8_wgrad_workspace_floats");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(dw, 16) || !aligned(db, 16) || !aligned(ws, 16))
    return invalid(what, "codes, scales, dw, db and workspace must be 16-byte aligned");
  if (!aligned(dy, es)) return invalid(what, "dy is not aligned to its elements");
  // a lane's offset from the step's first row, at most 24 rows and a width of 4 bytes, stays in 32 bits
  if (ld > (1 << 25)) return agpt_internal_set_error(AGPT_ERR_UNSUPPORTED, "agpt_act8: row strides above 2^25 are not supported");
  const Plan p = plan_of(T, out, in, shared_wo(out, in));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t n = static_cast<int64_t>(out) * in;
  const bool direct = p.chunks == 1;
  float* part = direct ? dw : ws;
  float* part_b = !db ? nullptr : (direct ? db : ws + static_cast<int64_t>(p.chunks) * n);
  const Grad g{T, ld, p.chunk_rows, out, in, p.tiles_o, p.tiles_i, p.chunks, relu ? 0.0f : 128.0f};
  const int64_t units = static_cast<int64_t>(p.chunks) * p.tiles_o * p.tiles_i;
  const dim3 grid(static_cast<unsigned>((units + kThreads / 64 - 1) / (kThreads / 64)));
  auto go = [&](auto e, auto pc, auto rc) {
    using E = decltype(e);
    hipLaunchKernelGGL((wgrad_kernel<E, decltype(pc)::value, decltype(rc)::value>), grid, dim3(kThreads), 0, st,
                       static_cast<const E*>(dy), hc, static_cast<E*>(dh), codes, scales, part, part_b, p.db_ld, g);
  };
  auto shared = [&](auto e, auto wc, auto rc) {
    using E = decltype(e);
    const int n = static_cast<int>((units + 7) / 8 * 8);
    hipLaunchKernelGGL((wgrad_shared_kernel<E, decltype(wc)::value, decltype(rc)::value>), dim3(n), dim3(kShared), 0, st,
                       static_cast<const E*>(dy), hc, static_cast<E*>(dh), codes, scales, part, part_b, p.db_ld, g, n);
  };
  using W2 = std::integral_constant<int, 2>;
  using W4 = std::integral_constant<int, 4>;
  auto kinds = [&](auto e) {
    if (p.wo == 2 && hc) shared(e, W2{}, std::true_type{});
    else if (p.wo == 2) shared(e, W2{}, std::false_type{});
    else if (p.wo == 4 && hc) shared(e, W4{}, std::true_type{});
    else if (p.wo == 4) shared(e, W4{}, std::false_type{});
    else if (hc) go(e, std::true_type{}, std::true_type{});
    else if (out > 1) go(e, std::true_type{}, std::false_type{});
    else go(e, std::false_type{}, std::false_type{});
  };
  if (dtype == AGPT_DTYPE_F32) kinds(float{});
  else kinds(bf16_t{});
  if (const int rc = launch_status(what)) return rc;
  if (direct) return AGPT_OK;
  if (n >= kAddWidth && p.chunks <= kAddChunks) {
    const int wblocks = static_cast<int>((n / 4 + kThreads - 1) / kThreads), bblocks = db ? (out + kThreads - 1) / kThreads : 0;
    hipLaunchKernelGGL(wgrad_add_kernel, dim3(wblocks + bblocks), dim3(kThreads), 0, st, part, n, part_b, p.db_ld, p.chunks,
                       out, dw, db, wblocks);
    return launch_status(what);
  }
  const int wblocks = static_cast<int>((n + 63) / 64), bblocks = db ? (out + 63) / 64 : 0;
  hipLaunchKernelGGL(wgrad_fold_kernel, dim3(wblocks + bblocks), dim3(kFoldThreads), 0, st, part, n, part_b, p.db_ld,
                     p.chunks, out, dw, db, wblocks);
  return launch_status(what);
}

}  // namespace

extern "C" int64_t agpt_act8_code_bytes(int64_t T, int W) { return T < 0 || W < 1 ? 0 : row_blocks(T) * kRows * W; }
extern "C" int64_t agpt_act8_scale_bytes(int64_t T, int W) {
  return T < 0 || W < 1 ? 0 : row_blocks(T) * kRows * (W / kBlock);
}

extern "C" int agpt_act8_pack(const void* x, int64_t ld_x, int dtype, int relu, uint8_t* codes, uint8_t* scales, int64_t T,
                              int W, void* stream) {
  const char* what = "agpt_act8_pack";
  if (const int rc = check(what, T, ld_x, W, W, dtype)) return rc;
  if (T == 0) return AGPT_OK;
  if (!x || !codes || !scales) return invalid(what, "null pointer");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(codes, 16) || !aligned(scales, 16)) return invalid(what, "codes and scales must be 16-byte aligned");
  if (!aligned(x, es)) return invalid(what, "x is not aligned to its elements");
  auto go = [&](auto e, auto vc) {
    using E = decltype(e);
    constexpr int V = decltype(vc)::value;
    const int pieces = W / (V == 1 ? 4 : V);
    const int64_t items = row_blocks(T) * pieces;
    const int gx = grid_of(items);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(gx), dim3(kThreads), 0, static_cast<hipStream_t>(stream), static_cast<const E*>(x),
                         ld_x, codes, scales, T, pieces, items, gx);
    };
    if (relu) launch(pack_kernel<E, V, true>);
    else launch(pack_kernel<E, V, false>);
  };
  const bool wide = ld_x * es % 16 == 0 && aligned(x, 16);
  using W8 = std::integral_constant<int, 8>;
  using W4 = std::integral_constant<int, 4>;
  using W1 = std::integral_constant<int, 1>;
  if (dtype == AGPT_DTYPE_F32) wide ? go(float{}, W4{}) : go(float{}, W1{});
  else wide ? go(bf16_t{}, W8{}) : go(bf16_t{}, W1{});
  return launch_status(what);
}

extern "C" int agpt_act8_unpack(const uint8_t* codes, const uint8_t* scales, int relu, void* x, int64_t ld_x, int dtype,
                                int64_t T, int W, void* stream) {
  const char* what = "agpt_act8_unpack";
  if (const int rc = check(what, T, ld_x, W, W, dtype)) return rc;
  if (T == 0) return AGPT_OK;
  if (!x || !codes || !scales) return invalid(what, "null pointer");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(codes, 16) || !aligned(scales, 16)) return invalid(what, "codes and scales must be 16-byte aligned");
  if (!aligned(x, es)) return invalid(what, "x is not aligned to its elements");
  const int quads = W / 4;
  const int64_t items = row_blocks(T) * quads;
  const int gx = grid_of(items);
  const bool wide = ld_x % 4 == 0 && aligned(x, 4 * es);
  auto go = [&](auto e, auto vc) {
    using E = decltype(e);
    hipLaunchKernelGGL((unpack_kernel<E, decltype(vc)::value>), dim3(gx), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                       codes, scales, static_cast<E*>(x), ld_x, T, quads, items, gx, relu ? 0.0f : 128.0f);
  };
  using W4 = std::integral_constant<int, 4>;
  using W1 = std::integral_constant<int, 1>;
  if (dtype == AGPT_DTYPE_F32) wide ? go(float{}, W4{}) : go(float{}, W1{});
  else wide ? go(bf16_t{}, W4{}) : go(bf16_t{}, W1{});
  return launch_status(what);
}

// One partial dW and db per chunk.
extern "C" int64_t agpt_act8_wgrad_workspace_floats(int64_t T, int out_width, int in_width) {
  if (T < 0 || out_width < 1 || in_width < 1) return 0;
  const Plan p = plan_of(T, out_width, in_width, shared_wo(out_width, in_width));
  return p.chunks * (static_cast<int64_t>(out_width) * in_width + p.db_ld);
}

extern "C" int agpt_act8_wgrad(const void* dy, int64_t ld_dy, int dtype, const uint8_t* codes, const uint8_t* scales,
                               int relu, float* dw, float* db, float* workspace, int64_t workspace_floats, int64_t T,
                               int out_width, int in_width, void* stream) {
  return wgrad("agpt_act8_wgrad", dy, ld_dy, dtype, nullptr, nullptr, codes, scales, relu, dw, db, workspace,
               workspace_floats, T, out_width, in_width, stream);
}

extern "C" int agpt_act8_relu_wgrad(const void* dh_in, int64_t ld_dh_in, int dtype, const uint8_t* h_codes, void* dh,
                                    const uint8_t* codes, const uint8_t* scales, int relu, float* dw, float* db,
                                    float* workspace, int64_t workspace_floats, int64_t T, int out_width, int in_width,
                                    void* stream) {
  const char* what = "agpt_act8_relu_wgrad";
  if (const int rc = check(what, T, ld_dh_in, out_width, out_width, dtype)) return rc;
  if (T > 0 && (!h_codes || !dh || !dh_in)) return invalid(what, "null pointer");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(dh_in, 16) || !aligned(dh, 16) || !aligned(h_codes, 16) || ld_dh_in * es % 16 != 0)
    return invalid(what, "dh_in, dh and h_codes must be 16-byte aligned, rows of dh_in too");
  if (T > 0 && dh == dh_in) return invalid(what, "dh must not overlap dh_in");
  return wgrad(what, dh_in, ld_dh_in, dtype, T > 0 ? h_codes : nullptr, dh, codes, scales, relu, dw, db, workspace,
               workspace_floats, T, out_width, in_width, stream);
}
