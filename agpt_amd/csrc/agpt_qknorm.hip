// agpt_qknorm.hip — the projection epilogue with a norm of every query and
// key head: bias, RMSNorm over the head, RoPE and the split into q, k, v in
// one pass, and its gradient in one pass (gfx950).
//
// With u = x (+ bias), per head of q and k, over its hd elements:
//   r = 1 / sqrt(mean(u^2) + eps),  y = u r w,  z = rotation(pos) y;  v = u.
//   g = rotation^T dz,  dw += g u r,  h = g w,  du = r (h - u r mean(h u r)).
// Both are HBM-bound: a head's L = hd / V lanes hold it in registers (V
// elements = 16 bytes each), so x (and dz) are read once and the results
// written once; r is recomputed in the backward, which reads x anyway.
//
// A thread keeps its column for all its rows, so the norm weights, the bias
// and the sums of dw and dbias stay in registers. Workgroups hold rpb whole
// rows (or, for wide rows, part of the heads of one: grid y), and walk the
// rows grid-strided. dw and dbias leave as one partial row per workgroup and
// are folded in a fixed order.
//
// 2^20 rows of 8 + 16 heads x 16 fp32: forward 600 us (3.2 GB at 5.4 TB/s), backward
// 845 + 11 (4.8 GB at 5.7); 32K rows of 32 + 16 heads x 128 bf16: backward 232 + 14
// (1.2 GB at 5.2 TB/s).

#include "rows.h"
#include "../../include/agpt_block.h"

#include <type_traits>

namespace {

using namespace agpt_rows;

constexpr int kMaxThreads = 512;
constexpr int kMaxGroupsX = 2048;  // workgroups (and partial rows of dw, dbias)

struct Shape {
  int64_t T, ld;  // rows, row stride of qkv and dqkv in elements
  int H, Hk, hd, seq;
  int S, Sp, rpb, gx, ny;  // head slots of a row, lane groups that a row takes, rows a workgroup holds, grid
  float eps;
};

// The head slot of this thread's group, its row within the workgroup's rows.
struct Place {
  int s, ro, col;
  bool row, live;  // the group has a slot; the lane has columns of it
};
template <int V, int L>
__device__ __forceinline__ Place place(const Shape& d, int threads) {
  const int tid = thread_x(), g = tid / L, groups = threads / L;
  Place p;
  if (d.ny > 1) {
    p.ro = 0;
    p.s = block_y() * groups + g;
    p.row = p.s < d.S;
  } else {
    p.ro = g / d.Sp;
    p.s = g - p.ro * d.Sp;
    p.row = p.ro < d.rpb && p.s < d.S;
  }
  p.col = (tid % L) * V;
  p.live = p.row && p.col < d.hd;
  return p;
}

// A row's cos and sin: cos(i), sin(i) of the pair (2i, 2i + 1), from table rows
// that hold each value twice. Where a head takes 16 lanes or more, a wave's lanes
// are all in one row: the wave fetches the row's tables once, a 16-byte load a
// lane, and hands the pairs out through its own part of LDS (each lane fetching
// its 64 bytes by itself kept the load units 81 % busy at 48 heads x 128 bf16).
template <int V, int L>
struct Turn {
  static constexpr bool kWave = L >= 16;
  static constexpr int kQuads = L * V > 128 ? 2 : 1;
  float4 q[kWave ? kQuads : 2 * (V / 4)];
  __device__ __forceinline__ void load(const float* __restrict__ cos_t, const float* __restrict__ sin_t, int p, int hd,
                                       int col) {
    const float* c = cos_t + static_cast<int64_t>(p) * hd;
    const float* s = sin_t + static_cast<int64_t>(p) * hd;
    if constexpr (kWave) {
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int i = (thread_x() & 63) + 64 * k, n = hd / 4;
        if (i < 2 * n) q[k] = *reinterpret_cast<const float4*>(i < n ? c + 4 * i : s + 4 * (i - n));
      }
    } else {
#pragma unroll
      for (int k = 0; k < V / 4; ++k) {
        q[2 * k] = *reinterpret_cast<const float4*>(c + col + 4 * k);
        q[2 * k + 1] = *reinterpret_cast<const float4*>(s + col + 4 * k);
      }
    }
  }
  // mine: the wave's 256 floats of LDS
  __device__ __forceinline__ void get(float* mine, int hd, int col, bool live, float (&c)[V / 2], float (&s)[V / 2]) const {
    if constexpr (kWave) {
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int i = (thread_x() & 63) + 64 * k;
        if (i < hd / 2) *reinterpret_cast<float2*>(mine + 2 * i) = float2{q[k].x, q[k].z};
      }
      __builtin_amdgcn_wave_barrier();
      if (live) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          c[i] = mine[col / 2 + i];
          s[i] = mine[hd / 2 + col / 2 + i];
        }
      }
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int k = 0; k < V / 4; ++k) {
        c[2 * k] = q[2 * k].x;
        c[2 * k + 1] = q[2 * k].z;
        s[2 * k] = q[2 * k + 1].x;
        s[2 * k + 1] = q[2 * k + 1].z;
      }
    }
  }
};
constexpr int kTabs = kMaxThreads / 64 * 256;

__device__ __forceinline__ int position_of(const int32_t* __restrict__ pos, bool turns, int64_t t, const Shape& d) {
  const int p = turns && t < d.T ? pos[t] : 0;
  return p < 0 ? 0 : (p > d.seq - 1 ? d.seq - 1 : p);
}

// Works on rows first, first + stride, ... below T. A row is worked on while the
// next one's elements and table rows are on their way, and the position of the
// one after it: the table rows wait for the position, and without that
// lead each row waits for both (32K rows of 48 heads x 128 bf16, backward: 437 -> 361 us).
template <typename Row, typename Position, typename Load, typename Work>
__device__ __forceinline__ void walk(int64_t first, int64_t stride, int64_t T, Position&& position, Load&& load,
                                     Work&& work) {
  Row r0, r1;
  int p1 = position(first + stride);
  load(first, position(first), r0);
  for (int64_t t = first; t < T; t += 2 * stride) {
    const int p2 = position(t + 2 * stride);
    load(t + stride, p1, r1);
    work(t, r0);
    if (t + stride >= T) break;
    p1 = position(t + 3 * stride);
    load(t + 2 * stride, p2, r0);
    work(t + stride, r1);
  }
}

template <typename T, int V, int L>
__global__ __launch_bounds__(kMaxThreads) void qk_fwd_kernel(const T* __restrict__ x, const float* __restrict__ bias,
                                                             const float* __restrict__ wq,
                                                             const float* __restrict__ wk,
                                                             const int32_t* __restrict__ pos,
                                                             const float* __restrict__ cos_t,
                                                             const float* __restrict__ sin_t, T* __restrict__ q,
                                                             T* __restrict__ k, T* __restrict__ v, Shape d,
                                                             int threads) {
  const Place me = place<V, L>(d, threads);
  const bool norm = me.s < d.H + d.Hk;
  float w[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = b[i] = 0.0f;
  if (me.live) {
    if (norm) load_row<V>((me.s < d.H ? wq : wk) + me.col, w);
    if (bias != nullptr) load_row<V>(bias + me.s * d.hd + me.col, b);
  }
  T* out = me.s < d.H ? q : (norm ? k : v);
  const int heads = me.s < d.H ? d.H : d.Hk;
  const int slot = me.s < d.H ? me.s : (norm ? me.s - d.H : me.s - d.H - d.Hk);
  const int64_t ostride = static_cast<int64_t>(heads) * d.hd, ooff = static_cast<int64_t>(slot) * d.hd + me.col;
  const int64_t xoff = static_cast<int64_t>(me.s) * d.hd + me.col;
  __shared__ float tabs[Turn<V, L>::kWave ? kTabs : 1];
  float* mine = tabs + (Turn<V, L>::kWave ? thread_x() / 64 * 256 : 0);
  const float inv = 1.0f / static_cast<float>(d.hd);
  // whether this lane's head turns; whether it fetches a table (in a wave of one row: for its neighbours too)
  const bool turns = norm && me.live && cos_t != nullptr, fetches = Turn<V, L>::kWave ? __ballot(turns) != 0 : turns;
  if (!me.row && !Turn<V, L>::kWave) return;
  const int64_t stride = static_cast<int64_t>(d.gx) * d.rpb, first = static_cast<int64_t>(block_x()) * d.rpb + me.ro;
  auto position = [&](int64_t t) { return position_of(pos, fetches, t, d); };
  struct Row {
    Raw<T, V> u;
    Turn<V, L> turn;
  };
  auto load = [&](int64_t t, int p, Row& r) {
    if (t >= d.T) return;
    if (me.live) r.u.load(x + t * d.ld + xoff);
    if (fetches) r.turn.load(cos_t, sin_t, p, d.hd, me.col);
  };
  auto work = [&](int64_t t, const Row& r) {
    float u[V], c[V / 2], s[V / 2];
    if (fetches) r.turn.get(mine, d.hd, me.col, turns, c, s);
#pragma unroll
    for (int i = 0; i < V; ++i) u[i] = 0.0f;
    if (me.live) r.u.get(u);
#pragma unroll
    for (int i = 0; i < V; ++i) u[i] += b[i];
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) ss += u[i] * u[i];
      const float q = __builtin_amdgcn_rsqf(lanes_sum<L>(ss) * inv + d.eps);
#pragma unroll
      for (int i = 0; i < V; ++i) u[i] = u[i] * q * w[i];
      if (turns) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float y0 = u[2 * i], y1 = u[2 * i + 1];
          u[2 * i] = y0 * c[i] - y1 * s[i];
          u[2 * i + 1] = y0 * s[i] + y1 * c[i];
        }
      }
    }
    if (me.live) store_row<V>(out + t * ostride + ooff, u);
  };
  walk<Row>(first, stride, d.T, position, load, work);
}

template <typename T, int V, int L>
__global__ __launch_bounds__(kMaxThreads) void qk_bwd_kernel(
    const T* __restrict__ dq, const T* __restrict__ dk, const T* __restrict__ dv, const T* __restrict__ x,
    const float* __restrict__ bias, const float* __restrict__ wq, const float* __restrict__ wk,
    const int32_t* __restrict__ pos, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    T* __restrict__ dx, int64_t ld_dx, float* __restrict__ part_w, float* __restrict__ part_b, Shape d, int threads) {
  __shared__ float red[kMaxThreads * V];
  const Place me = place<V, L>(d, threads);
  const bool norm = me.s < d.H + d.Hk;
  float w[V], b[V], dw[V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = b[i] = dw[i] = db[i] = 0.0f;
  if (me.live) {
    if (norm) load_row<V>((me.s < d.H ? wq : wk) + me.col, w);
    if (bias != nullptr) load_row<V>(bias + me.s * d.hd + me.col, b);
  }
  const T* dz = me.s < d.H ? dq : (norm ? dk : dv);
  const int heads = me.s < d.H ? d.H : d.Hk;
  const int slot = me.s < d.H ? me.s : (norm ? me.s - d.H : me.s - d.H - d.Hk);
  const int64_t zstride = static_cast<int64_t>(heads) * d.hd, zoff = static_cast<int64_t>(slot) * d.hd + me.col;
  const int64_t xoff = static_cast<int64_t>(me.s) * d.hd + me.col;
  const float inv = 1.0f / static_cast<float>(d.hd);
  __shared__ float tabs[Turn<V, L>::kWave ? kTabs : 1];
  float* mine = tabs + (Turn<V, L>::kWave ? thread_x() / 64 * 256 : 0);
  // whether this lane's head turns; whether it fetches a table (in a wave of one row: for its neighbours too)
  const bool turns = norm && me.live && cos_t != nullptr, fetches = Turn<V, L>::kWave ? __ballot(turns) != 0 : turns;
  if (me.row || Turn<V, L>::kWave) {
    const int64_t stride = static_cast<int64_t>(d.gx) * d.rpb;
    const int64_t first = static_cast<int64_t>(block_x()) * d.rpb + me.ro;
    auto position = [&](int64_t t) { return position_of(pos, fetches, t, d); };
    struct Row {
      Raw<T, V> g, u;
      Turn<V, L> turn;
    };
    auto load = [&](int64_t t, int p, Row& r) {
      if (t >= d.T) return;
      if (me.live) {
        r.g.load(dz + t * zstride + zoff);
        if (norm) r.u.load(x + t * d.ld + xoff);
      }
      if (fetches) r.turn.load(cos_t, sin_t, p, d.hd, me.col);
    };
    auto work = [&](int64_t t, const Row& r) {
      float g[V], u[V], c[V / 2], s[V / 2];
      if (fetches) r.turn.get(mine, d.hd, me.col, turns, c, s);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = u[i] = 0.0f;
      if (me.live) r.g.get(g);
      if (norm) {
        if (me.live) r.u.get(u);
        if (turns) {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const float z0 = g[2 * i], z1 = g[2 * i + 1];
            g[2 * i] = z0 * c[i] + z1 * s[i];
            g[2 * i + 1] = z1 * c[i] - z0 * s[i];
          }
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          u[i] += b[i];
          ss += u[i] * u[i];
        }
        const float q = __builtin_amdgcn_rsqf(lanes_sum<L>(ss) * inv + d.eps);
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          u[i] *= q;
          dw[i] += g[i] * u[i];
          g[i] *= w[i];
          m += g[i] * u[i];
        }
        m = lanes_sum<L>(m) * inv;
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = q * (g[i] - u[i] * m);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) db[i] += g[i];
      if (me.live) store_row<V>(dx + t * ld_dx + xoff, g);
    };
    walk<Row>(first, stride, d.T, position, load, work);
  }
  // dbias of the workgroup's columns: its rows of a slot added in row order
  const int tid = thread_x(), groups = threads / L, first = d.ny > 1 ? block_y() * groups : 0;
  const int slots = d.ny > 1 ? (d.S - first < groups ? d.S - first : groups) : d.S;
  constexpr int W = L * V;
  if (part_b != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) red[tid * V + i] = db[i];
    __syncthreads();
    for (int j = tid; j < slots * d.hd; j += threads) {
      const int s = j / d.hd, c = j - s * d.hd;
      float a = 0.0f;
      for (int o = 0; o < d.rpb; ++o) a += red[(o * d.Sp + s) * W + c];
      part_b[(static_cast<int64_t>(block_x()) * d.S + first) * d.hd + j] = a;
    }
    __syncthreads();
  }
  // dw of its query heads, then of its key heads, in slot and row order
#pragma unroll
  for (int i = 0; i < V; ++i) red[tid * V + i] = dw[i];
  __syncthreads();
  for (int j = tid; j < 2 * d.hd; j += threads) {
    const int key = j >= d.hd, c = j - key * d.hd;
    const int lo = key ? d.H : 0, hi = key ? d.H + d.Hk : d.H;
    float a = 0.0f;
    for (int o = 0; o < d.rpb; ++o)
      for (int s = 0; s < slots; ++s)
        if (first + s >= lo && first + s < hi) a += red[(o * d.Sp + s) * W + c];
    part_w[(static_cast<int64_t>(block_x()) * d.ny + block_y()) * 2 * d.hd + j] = a;
  }
}

// dwq | dwk from the partial rows of every workgroup, dbias from those of its columns.
__global__ __launch_bounds__(kFoldThreads) void qk_fold_kernel(const float* __restrict__ part_w,
                                                               const float* __restrict__ part_b,
                                                               float* __restrict__ dwq, float* __restrict__ dwk,
                                                               float* __restrict__ db, int gx, int ny, int hd, int C,
                                                               int wblocks) {
  const int blk = block_x();
  if (blk < 2 * wblocks) {
    const int key = blk >= wblocks;
    fold_columns(part_w + key * hd, 2 * hd, gx * ny, hd, blk - key * wblocks, key ? dwk : dwq);
  } else {
    fold_columns(part_b, C, gx, C, blk - 2 * wblocks, db);
  }
}

struct Launch {
  int threads, V, L;
};

// The launch shape: L lanes to a head; the workgroup size whose lanes whole
// rows fill best (24 heads of 16: 192 threads hold two rows, 256 would leave
// a quarter idle), or 256 threads over part of a wide row's heads.
Launch shape_of(Shape& d, bool bf16) {
  Launch l;
  l.V = bf16 && d.hd % 8 == 0 ? 8 : 4;
  l.L = 1;
  while (l.L * l.V < d.hd) l.L *= 2;
  d.S = d.H + 2 * d.Hk;
  const int pad = l.L >= 16 ? 64 / l.L : 1;  // whole waves to a row, as Turn takes it
  d.Sp = (d.S + pad - 1) / pad * pad;
  const int row = d.Sp * l.L;
  l.threads = 256;
  if (row > kMaxThreads) {
    d.rpb = 1;
    d.ny = (row + 255) / 256;
  } else {
    static const int kSizes[] = {256, 192, 128, 320, 384, 448, 512};
    double best = -1.0;
    for (const int n : kSizes) {
      const double use = static_cast<double>(n / row * row) / n;
      if (use > best + 1e-9) {
        best = use;
        l.threads = n;
      }
    }
    d.rpb = l.threads / row;
    d.ny = 1;
  }
  const int64_t need = (d.T + d.rpb - 1) / d.rpb;
  const int cap = kMaxGroupsX / d.ny > 0 ? kMaxGroupsX / d.ny : 1;
  d.gx = static_cast<int>(need < cap ? need : cap);
  return l;
}

template <typename T, int V, typename Fn>
bool with_lanes(int L, Fn&& fn) {
  switch (L) {
    case 1: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 1>{}); return true;
    case 2: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 2>{}); return true;
    case 4: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 4>{}); return true;
    case 8: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 8>{}); return true;
    case 16: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 16>{}); return true;
    case 32: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 32>{}); return true;
    case 64: fn(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 64>{}); return true;
    default: return false;
  }
}
template <typename Fn>
bool with_kernel(const Launch& l, int dtype, Fn&& fn) {
  if (dtype == AGPT_DTYPE_F32) return with_lanes<float, 4>(l.L, fn);
  if (l.V == 8) return with_lanes<bf16_t, 8>(l.L, fn);
  return with_lanes<bf16_t, 4>(l.L, fn);
}

int check_shape(const char* what, int64_t T, int64_t ld, int n_heads, int n_kv_heads, int head_dim, int dtype,
                bool rope, int seq, int64_t C, float eps) {
  if (T < 0 || n_heads < 1 || n_kv_heads < 1) return invalid(what, "T < 0, n_heads < 1 or n_kv_heads < 1");
  if (head_dim < 4 || head_dim > 256 || head_dim % 4 != 0) {
    char msg[160];
    snprintf(msg, sizeof(msg), "%s: head_dim must be a multiple of 4 from 4 to 256 (got %d)", what, head_dim);
    return agpt_internal_set_error(AGPT_ERR_UNSUPPORTED, msg);
  }
  if (n_heads > 65536 / head_dim || n_kv_heads > 65536 / head_dim)
    return invalid(what, "a row of more than 65536 query or key elements");
  if (dtype != AGPT_DTYPE_F32 && dtype != AGPT_DTYPE_BF16) return invalid(what, "unknown dtype");
  if (ld < C) return invalid(what, "row stride smaller than a row");
  if (ld % (dtype == AGPT_DTYPE_BF16 && head_dim % 8 == 0 ? 8 : 4) != 0)
    return invalid(what, "row stride must be a multiple of 4 elements (of 8 in bf16 where head_dim is)");
  if (rope && seq < 1) return invalid(what, "rope_seq_len < 1");
  if (!(eps >= 0.0f)) return invalid(what, "eps must not be negative");
  return AGPT_OK;
}

}  // namespace

extern "C" int agpt_qk_norm_rope_split(const void* qkv, int64_t ld_qkv, const float* bias, const float* wq,
                                       const float* wk, const int32_t* positions, const float* cos_t,
                                       const float* sin_t, int rope_seq_len, int64_t T, int n_heads, int n_kv_heads,
                                       int head_dim, float eps, int dtype, void* q, void* k, void* v, void* stream) {
  const char* what = "agpt_qk_norm_rope_split";
  const int64_t C = (static_cast<int64_t>(n_heads) + 2 * static_cast<int64_t>(n_kv_heads)) * head_dim;
  if (const int rc = check_shape(what, T, ld_qkv, n_heads, n_kv_heads, head_dim, dtype, cos_t != nullptr, rope_seq_len, C,
                               eps))
    return rc;
  if (T == 0) return AGPT_OK;
  if (!qkv || !wq || !wk || !q || !k || !v || (cos_t && (!sin_t || !positions)))
    return invalid(what, "null pointer");
  for (const void* p : {qkv, static_cast<const void*>(bias), static_cast<const void*>(wq), static_cast<const void*>(wk),
                        static_cast<const void*>(cos_t), static_cast<const void*>(sin_t), static_cast<const void*>(q),
                        static_cast<const void*>(k), static_cast<const void*>(v)})
    if (!aligned(p, 16)) return invalid(what, "buffers must be 16-byte aligned");
  Shape d{T, ld_qkv, n_heads, n_kv_heads, head_dim, rope_seq_len, 0, 0, 0, 0, 0, eps};
  const Launch l = shape_of(d, dtype == AGPT_DTYPE_BF16);
  with_kernel(l, dtype, [&](auto t, auto vc, auto lc) {
    using E = decltype(t);
    hipLaunchKernelGGL((qk_fwd_kernel<E, decltype(vc)::value, decltype(lc)::value>), dim3(d.gx, d.ny), dim3(l.threads), 0,
                       static_cast<hipStream_t>(stream), static_cast<const E*>(qkv), bias, wq, wk, positions, cos_t,
                       sin_t, static_cast<E*>(q), static_cast<E*>(k), static_cast<E*>(v), d, l.threads);
  });
  return launch_status(what);
}

// Floats of the partial rows: gx * ny rows of 2 hd, gx rows of C.
extern "C" int64_t agpt_qk_norm_workspace_floats(int n_heads, int n_kv_heads, int head_dim) {
  if (n_heads < 1 || n_kv_heads < 1 || head_dim < 1) return 0;
  const int64_t C = (static_cast<int64_t>(n_heads) + 2 * static_cast<int64_t>(n_kv_heads)) * head_dim;
  return static_cast<int64_t>(kMaxGroupsX) * (2 * head_dim + C);
}

extern "C" int agpt_qk_norm_rope_split_bwd(const void* dq, const void* dk, const void* dv, const void* qkv,
                                           int64_t ld_qkv, const float* bias, const float* wq, const float* wk,
                                           const int32_t* positions, const float* cos_t, const float* sin_t,
                                           int rope_seq_len, int64_t T, int n_heads, int n_kv_heads, int head_dim,
                                           float eps, int dtype, void* dqkv, int64_t ld_dqkv, float* dwq, float* dwk,
                                           float* dbias, float* workspace, int64_t workspace_floats, void* stream) {
  const char* what = "agpt_qk_norm_rope_split_bwd";
  const int64_t C = (static_cast<int64_t>(n_heads) + 2 * static_cast<int64_t>(n_kv_heads)) * head_dim;
  for (const int64_t ld : {ld_qkv, ld_dqkv})
    if (const int rc = check_shape(what, T, ld, n_heads, n_kv_heads, head_dim, dtype, cos_t != nullptr, rope_seq_len, C,
                               eps))
      return rc;
  if (!wq || !wk || !dwq || !dwk || !workspace ||
      (T > 0 && (!dq || !dk || !dv || !qkv || !dqkv || (cos_t && (!sin_t || !positions)))))
    return invalid(what, "null pointer");
  if (workspace_floats < agpt_qk_norm_workspace_floats(n_heads, n_kv_heads, head_dim))
    return invalid(what, "workspace smaller than agpt_qk_norm_workspace_floats");
  for (const void* p : {dq, dk, dv, qkv, static_cast<const void*>(bias), static_cast<const void*>(wq),
                        static_cast<const void*>(wk), static_cast<const void*>(cos_t), static_cast<const void*>(sin_t),
                        static_cast<const void*>(dqkv), static_cast<const void*>(dwq), static_cast<const void*>(dwk),
                        static_cast<const void*>(dbias), static_cast<const void*>(workspace)})
    if (!aligned(p, 16)) return invalid(what, "buffers must be 16-byte aligned");
  Shape d{T, ld_qkv, n_heads, n_kv_heads, head_dim, rope_seq_len, 0, 0, 0, 0, 0, eps};
  const Launch l = shape_of(d, dtype == AGPT_DTYPE_BF16);
  if (d.gx < 1) d.gx = 1;  // no rows: the sums are zeros
  float* part_w = workspace;
  float* part_b = workspace + static_cast<int64_t>(d.gx) * d.ny * 2 * head_dim;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  with_kernel(l, dtype, [&](auto t, auto vc, auto lc) {
    using E = decltype(t);
    hipLaunchKernelGGL((qk_bwd_kernel<E, decltype(vc)::value, decltype(lc)::value>), dim3(d.gx, d.ny), dim3(l.threads), 0, st,
                       static_cast<const E*>(dq), static_cast<const E*>(dk), static_cast<const E*>(dv),
                       static_cast<const E*>(qkv), bias, wq, wk, positions, cos_t, sin_t, static_cast<E*>(dqkv), ld_dqkv,
                       part_w, dbias ? part_b : nullptr, d, l.threads);
  });
  if (const int rc = launch_status(what)) return rc;
  const int wblocks = (head_dim + 63) / 64, bblocks = dbias ? static_cast<int>((C + 63) / 64) : 0;
  hipLaunchKernelGGL(qk_fold_kernel, dim3(2 * wblocks + bblocks), dim3(kFoldThreads), 0, st, part_w, part_b, dwq, dwk,
                     dbias, d.gx, d.ny, head_dim, static_cast<int>(C), wblocks);
  return launch_status(what);
}
