// agpt_embed.hip — the token embedding (gfx950): x = scale * E[token], and
// dE[v] = scale * (sum of dx over the rows of token v) with the rows sorted by
// token, so that each sum has one owner and a fixed order and no row of dE is
// added to by two workgroups.
//
// Sort: a stable counting sort of (token, row) by digits of up to 8 bits, low
// digit first: per tile of 2048 rows a digit histogram, per digit a scan over
// the tiles, then each tile places its rows by ballots (equal digits of a wave
// keep their lane order, waves their order through per-wave counts).
//
// Sums: the sorted rows are cut into spans of R. A token of up to R rows is
// summed by one wave that gathers its rows; a longer one is summed piecewise,
// at most two pieces per span (the end of one long token and the start of the
// next), and its pieces are added in span order.

#include "rows.h"
#include "../../include/agpt_embed.h"

#include <type_traits>

namespace {

using namespace agpt_rows;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ---- lookup ------------------------------------------------------------------
// `lanes` threads (a power of two) hold a row in pieces of V elements; a
// workgroup takes kThreads / lanes rows at a time.
template <typename T, typename I, int V>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(const T* __restrict__ table, const I* __restrict__ tokens,
                                                             float scale, T* __restrict__ x, int64_t rows, int64_t vocab,
                                                             int D, int lanes, int gx) {
  const int tid = thread_x(), c0 = (tid & (lanes - 1)) * V, rpb = kThreads / lanes;
  for (int64_t t = static_cast<int64_t>(block_x()) * rpb + tid / lanes; t < rows; t += static_cast<int64_t>(gx) * rpb) {
    const int64_t tok = static_cast<int64_t>(tokens[t]);
    const bool ok = tok >= 0 && tok < vocab;
    for (int c = c0; c < D; c += lanes * V) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = 0.0f;
      if (ok) load_row<V>(table + tok * D + c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = ok ? v[i] * scale : 0.0f;
      store_row<V>(x + t * D + c, v);
    }
  }
}

// ---- sort ----------------------------------------------------------------------
constexpr int kTile = 2048;      // rows of a sort tile, kTile / kWaves of them per wave
constexpr int kMaxBits = 8;      // digit width
constexpr int kDigits = 1 << kMaxBits;

// The sort key: the token, or V for padding.
template <typename I>
__device__ __forceinline__ int32_t key_of(I token, int64_t vocab) {
  const int64_t t = static_cast<int64_t>(token);
  return static_cast<int32_t>(t >= 0 && t < vocab ? t : vocab);
}

// counts[digit][tile]. kFirst: keys come from the tokens.
template <typename I, bool kFirst>
__global__ __launch_bounds__(kThreads) void hist_kernel(const I* __restrict__ keys, int64_t n, int64_t vocab, int shift,
                                                        int digits, int32_t* __restrict__ counts, int tiles) {
  __shared__ int h[kDigits];
  const int tid = thread_x(), tile = block_x();
  h[tid] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(tile) * kTile;
#pragma unroll 4
  for (int i = tid; i < kTile; i += kThreads) {
    if (base + i < n) {
      const int32_t k = kFirst ? key_of(keys[base + i], vocab) : static_cast<int32_t>(keys[base + i]);
      atomicAdd(&h[(k >> shift) & (digits - 1)], 1);
    }
  }
  __syncthreads();
  if (tid < digits) counts[static_cast<int64_t>(tid) * tiles + tile] = h[tid];
}

// Inclusive sum over the workgroup's threads; `wsum` holds kWaves ints.
__device__ __forceinline__ int block_scan(int v, int* wsum) {
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  if (lane == 63) wsum[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += wsum[w];
  return v;
}

// One workgroup per digit: counts[digit][.] becomes its exclusive scan over
// the tiles, totals[digit] the digit's rows.
__global__ __launch_bounds__(kThreads) void scan_kernel(int32_t* __restrict__ counts, int tiles,
                                                        int32_t* __restrict__ totals) {
  __shared__ int wsum[kWaves];
  const int tid = thread_x();
  int32_t* row = counts + static_cast<int64_t>(block_x()) * tiles;
  int carry = 0;
  for (int a = 0; a < tiles; a += kThreads) {
    const int i = a + tid, v = i < tiles ? row[i] : 0;
    const int inc = block_scan(v, wsum);
    if (i < tiles) row[i] = carry + inc - v;
    int all = 0;
    for (int w = 0; w < kWaves; ++w) all += wsum[w];
    carry += all;
    __syncthreads();
  }
  if (tid == 0) totals[block_x()] = carry;
}

// Places a tile's rows: digit start + rows of the digit in earlier tiles +
// rank within the tile. kFirst: keys from the tokens, rows are 0, 1, .... offsets: where this is the only pass.
template <typename I, bool kFirst>
__global__ __launch_bounds__(kThreads) void place_kernel(const I* __restrict__ keys, const int32_t* __restrict__ rows,
                                                         int64_t n, int64_t vocab, int shift, int bits,
                                                         const int32_t* __restrict__ counts,
                                                         const int32_t* __restrict__ totals, int tiles,
                                                         int32_t* __restrict__ keys_out,
                                                         int32_t* __restrict__ rows_out,
                                                         int32_t* __restrict__ offsets) {
  __shared__ int next[kWaves][kDigits];  // where the wave's next row of a digit goes
  __shared__ int wsum[kWaves];
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6, tile = block_x(), digits = 1 << bits;
  for (int w = 0; w < kWaves; ++w) next[w][tid] = 0;
  __syncthreads();
  constexpr int kPerWave = kTile / kWaves, kRounds = kPerWave / 64;
  const int64_t base = static_cast<int64_t>(tile) * kTile + wave * kPerWave + lane;
  int32_t k[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 64;
    k[r] = i < n ? (kFirst ? key_of(keys[i], vocab) : static_cast<int32_t>(keys[i])) : 0;
    if (i < n) atomicAdd(&next[wave][(k[r] >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  {
    const int tot = tid < digits ? totals[tid] : 0;
    int at = block_scan(tot, wsum) - tot;
    // a single digit is the whole key: its starts are the plan's offsets
    if (offsets != nullptr && tile == 0 && tid <= vocab) offsets[tid] = at;
    if (tid < digits) {
      at += counts[static_cast<int64_t>(tid) * tiles + tile];
      for (int w = 0; w < kWaves; ++w) {
        const int c = next[w][tid];
        next[w][tid] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 64;
    const bool in = i < n;
    const int d = (k[r] >> shift) & (digits - 1);
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? set : ~set;
    }
    const int rank = __popcll(same & below);
    int at = 0;
    if (in) at = next[wave][d] + rank;
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) next[wave][d] = at + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (in) {
      keys_out[at] = k[r];
      rows_out[at] = kFirst ? static_cast<int32_t>(i) : rows[i];
    }
  }
}

// offsets[v] = the first sorted place whose key is not below v, v <= V.
__global__ __launch_bounds__(kThreads) void offsets_kernel(const int32_t* __restrict__ keys, int32_t n, int32_t vocab,
                                                           int32_t* __restrict__ offsets) {
  const int64_t v = static_cast<int64_t>(block_x()) * kThreads + thread_x();
  if (v > vocab) return;
  int32_t lo = 0, hi = n;
  while (lo < hi) {
    const int32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  offsets[v] = lo;
}

// ---- sums ----------------------------------------------------------------------
// Workgroups 0 .. spans - 1: the pieces of long tokens in their span, to
// part[2 span] (a token begun in an earlier span) and part[2 span + 1] (one
// that begins here and goes on past the span). The others: a wave per token
// of up to R rows, zeros where it has none.
template <typename T, int V>
__device__ __forceinline__ void gather_sum(const T* __restrict__ dx, int64_t ld, const int32_t* __restrict__ order,
                                           int a, int b, int step, int c, float (&s)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.0f;
#pragma unroll 8
  for (int j = a; j < b; j += step) {
    float v[V];
    load_row<V>(dx + order[j] * ld + c, v);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] += v[i];
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void sums_kernel(const T* __restrict__ dx, int64_t ld,
                                                        const int32_t* __restrict__ order,
                                                        const int32_t* __restrict__ keys,
                                                        const int32_t* __restrict__ offsets, float scale,
                                                        float* __restrict__ dE, float* __restrict__ part, int32_t n,
                                                        int32_t vocab, int D, int R, int spans, int lanes) {
  __shared__ float red[kThreads * V];
  const int tid = thread_x(), blk = block_x();
  if (blk < spans) {
    const int32_t s0 = blk * R, s1 = s0 + R < n ? s0 + R : n;
    const int32_t first = keys[s0], last = keys[s1 - 1];
    for (int piece = 0; piece < 2; ++piece) {
      const int32_t v = piece ? last : first;
      if (v >= vocab) continue;
      const int32_t a = offsets[v], b = offsets[v + 1];
      if (b - a <= R || (a < s0) != (piece == 0)) continue;
      const int32_t p0 = a > s0 ? a : s0, p1 = b < s1 ? b : s1;
      const int slots = kThreads / lanes, slot = tid / lanes;
      for (int c0 = 0; c0 < D; c0 += lanes * V) {
        const int c = c0 + (tid & (lanes - 1)) * V;
        float s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = 0.0f;
        if (c < D) gather_sum<T, V>(dx, ld, order, p0 + slot, p1, slots, c, s);
#pragma unroll
        for (int i = 0; i < V; ++i) red[tid * V + i] = s[i];
        __syncthreads();
        if (slot == 0 && c < D) {
          for (int q = 1; q < slots; ++q)
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += red[(q * lanes + tid) * V + i];
          float* out = part + (2 * static_cast<int64_t>(blk) + piece) * D + c;
#pragma unroll
          for (int i = 0; i < V; ++i) out[i] = s[i];
        }
        __syncthreads();
      }
    }
    return;
  }
  const int64_t v = static_cast<int64_t>(blk - spans) * kWaves + (tid >> 6);
  if (v >= vocab) return;
  const int32_t a = offsets[v], b = offsets[v + 1];
  if (b - a > R) return;
  for (int c = (tid & 63) * V; c < D; c += 64 * V) {
    float s[V];
    gather_sum<T, V>(dx, ld, order, a, b, 1, c, s);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= scale;
    store_row<V>(dE + v * D + c, s);
  }
}

// Workgroup `span`: the long token that begins in it and goes on past it, if
// there is one: its pieces, dealt to slots of `lanes` columns, the slots added in order.
constexpr int kJoin = 1024;
__global__ __launch_bounds__(kJoin) void join_kernel(const float* __restrict__ part, const int32_t* __restrict__ keys,
                                                     const int32_t* __restrict__ offsets, float scale,
                                                     float* __restrict__ dE, int32_t n, int32_t vocab, int D, int R,
                                                     int lanes) {
  __shared__ float red[kJoin];
  const int span = block_x(), tid = thread_x();
  const int32_t s0 = span * R, s1 = s0 + R < n ? s0 + R : n;
  const int32_t v = keys[s1 - 1];
  if (v >= vocab) return;
  const int32_t a = offsets[v], b = offsets[v + 1];
  if (b - a <= R || a < s0) return;
  const int end = (b - 1) / R, slots = kJoin / lanes, slot = tid / lanes;
  for (int c0 = 0; c0 < D; c0 += lanes) {
    const int c = c0 + (tid & (lanes - 1));
    float s = 0.0f;
    if (c < D) {
      if (slot == 0) s = part[(2 * static_cast<int64_t>(span) + 1) * D + c];
#pragma unroll 8
      for (int q = span + 1 + slot; q <= end; q += slots) s += part[2 * static_cast<int64_t>(q) * D + c];
    }
    red[tid] = s;
    __syncthreads();
    if (slot == 0 && c < D) {
      for (int q = 1; q < slots; ++q) s += red[q * lanes + tid];
      dE[static_cast<int64_t>(v) * D + c] = s * scale;
    }
    __syncthreads();
  }
}

// ---- one launch for short batches --------------------------------------------------
// A workgroup owns the tokens v = range (mod ranges), ranges a power of two (so
// that neighbouring, often equally frequent ids part), and 64 V columns. It reads
// every token of the batch from L2, lists the rows of its own, sorts the list
// (stable, by the token's number within the range: at most 256, one digit) and
// sums each token's rows, a wave per token; a token of many rows takes all waves.
constexpr int kDirect = 512, kDirectWaves = kDirect / 64;
constexpr int kLocal = 256;  // tokens of a range at most

template <typename T, typename I, int V, int kCap>
__global__ __launch_bounds__(kDirect) void direct_kernel(const T* __restrict__ dx, int64_t ld,
                                                         const I* __restrict__ tokens, float scale,
                                                         float* __restrict__ dE, int n, int64_t vocab, int D, int log_ranges,
                                                         int lanes) {
  __shared__ uint16_t found[kCap + kDirect], rows[kCap + kDirect];
  __shared__ int next[kDirectWaves][kLocal];
  __shared__ int start[kLocal + 1];
  __shared__ int wsum[kDirectWaves];
  __shared__ float red[kDirect * V];
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6, blk = block_x();
  const int ranges = 1 << log_ranges, range = blk & (ranges - 1), slice = blk >> log_ranges;
  const int per_range = static_cast<int>((vocab + ranges - 1) >> log_ranges);
  const uint64_t below = (1ull << lane) - 1;

  const int share = (n + kDirect - 1) / kDirect * 64, first = wave * share;
  const int last = first + share < n ? first + share : n;
  int cnt = 0;
  for (int i = first; i < last; i += 4 * 64) {
    I tok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) tok[u] = i + u * 64 + lane < last ? tokens[i + u * 64 + lane] : static_cast<I>(-1);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t t = static_cast<int64_t>(tok[u]);
      const bool mine = t >= 0 && t < vocab && (static_cast<int>(t) & (ranges - 1)) == range;
      const uint64_t m = __ballot(mine);
      if (mine) found[first + cnt + __popcll(m & below)] = static_cast<uint16_t>(i + u * 64 + lane);
      cnt += __popcll(m);
    }
  }
  for (int i = lane; i < kLocal; i += 64) next[wave][i] = 0;
  __builtin_amdgcn_wave_barrier();
  auto local_of = [&](int row) { return static_cast<int>(static_cast<int64_t>(tokens[row]) >> log_ranges); };
  for (int j = lane; j < cnt; j += 64) atomicAdd(&next[wave][local_of(found[first + j])], 1);
  __syncthreads();
  {
    int tot = 0;
    if (tid < kLocal)
      for (int w = 0; w < kDirectWaves; ++w) tot += next[w][tid];
    int inc = tot;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int u = __shfl_up(inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    for (int w = 0; w < wave; ++w) inc += wsum[w];
    if (tid < kLocal) {
      int at = inc - tot;
      start[tid] = at;
      if (tid == kLocal - 1) start[kLocal] = inc;
      for (int w = 0; w < kDirectWaves; ++w) {
        const int c = next[w][tid];
        next[w][tid] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  for (int j = 0; j < cnt; j += 64) {
    const bool in = j + lane < cnt;
    const int row = in ? found[first + j + lane] : 0;
    const int d = in ? local_of(row) : 0;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? set : ~set;
    }
    const int rank = __popcll(same & below);
    int at = 0;
    if (in) at = next[wave][d] + rank;
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) next[wave][d] = at + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (in) rows[at] = static_cast<uint16_t>(row);
  }
  __syncthreads();

  const int groups = 64 / lanes, grp = lane / lanes, c = slice * 64 * V + (lane & (lanes - 1)) * V;
  const int kLong = 64 * groups;  // rows that a wave sums by itself
  auto sum_rows = [&](int a, int b, float (&s)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.0f;
    if (c < D) {
#pragma unroll 8
      for (int j = a + grp; j < b; j += groups) {
        float x[V];
        load_row<V>(dx + rows[j] * ld + c, x);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += x[i];
      }
    }
    for (int o = lanes; o < 64; o *= 2)
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += __shfl_xor(s[i], o);
  };
  for (int k = wave; k < per_range; k += kDirectWaves) {
    const int64_t v = (static_cast<int64_t>(k) << log_ranges) | range;
    const int a = start[k], b = start[k + 1];
    if (v >= vocab || b - a > kLong) continue;
    float s[V];
    sum_rows(a, b, s);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= scale;
    if (grp == 0 && c < D) store_row<V>(dE + v * D + c, s);
  }
  for (int k = 0; k < per_range; ++k) {
    const int a = start[k], b = start[k + 1];
    if (b - a <= kLong) continue;
    const int64_t v = (static_cast<int64_t>(k) << log_ranges) | range;
    const int each = (b - a + kDirectWaves - 1) / kDirectWaves, w0 = a + wave * each;
    float s[V];
    sum_rows(w0 < b ? w0 : b, w0 + each < b ? w0 + each : b, s);
#pragma unroll
    for (int i = 0; i < V; ++i) red[tid * V + i] = s[i];
    __syncthreads();
    if (wave == 0 && grp == 0 && c < D) {
      for (int w = 1; w < kDirectWaves; ++w)
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += red[(w * 64 + lane) * V + i];
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] *= scale;
      store_row<V>(dE + v * D + c, s);
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kThreads) void zero_kernel(float* __restrict__ p, int64_t n, int gx) {
  for (int64_t i = static_cast<int64_t>(block_x()) * kThreads + thread_x(); i < n; i += static_cast<int64_t>(gx) * kThreads)
    p[i] = 0.0f;
}

constexpr int64_t kMaxCount = 0x7fffffff - 4096;  // places and steps past the last one stay in 32 bits

int digit_bits(int64_t V, int* passes) {
  int bits = 1;
  while ((V >> bits) != 0) ++bits;  // keys 0 .. V
  *passes = (bits + kMaxBits - 1) / kMaxBits;
  return (bits + *passes - 1) / *passes;
}

// Rows of a span: enough spans to fill the chip, few enough pieces to add.
int span_rows(int64_t T) {
  int R = 64;
  while (R < 512 && T / R > 2048) R *= 2;
  return R;
}

int64_t tiles_of(int64_t T) { return (T + kTile - 1) / kTile; }

int lanes_for(int D, int V) {
  int lanes = 1;
  while (lanes * V < D && lanes < kThreads) lanes *= 2;
  return lanes;
}

int check_counts(const char* what, int64_t T, int64_t V) {
  if (T < 0 || V < 1) return invalid(what, "T < 0 or V < 1");
  if (T > kMaxCount || V > kMaxCount) return invalid(what, "T and V must be below 2^31 - 4096");
  return AGPT_OK;
}

// Whether rows of dx and of the table go in 16-byte pieces.
bool wide_rows(int D, int64_t ld, int es, const void* dx, const void* table) {
  return static_cast<int64_t>(D) * es % 16 == 0 && ld * es % 16 == 0 && aligned(dx, 16) && aligned(table, 16);
}

template <typename Fn>
void with_dtype(int dtype, bool wide, Fn&& fn) {
  if (dtype == AGPT_DTYPE_F32) {
    if (wide) fn(float{}, std::integral_constant<int, 4>{});
    else fn(float{}, std::integral_constant<int, 1>{});
  } else {
    if (wide) fn(bf16_t{}, std::integral_constant<int, 8>{});
    else fn(bf16_t{}, std::integral_constant<int, 1>{});
  }
}

}  // namespace

extern "C" int agpt_embed_fwd(const void* table, const void* tokens, int token_bits, float scale, void* x, int64_t T,
                              int64_t V, int D, int dtype, void* stream) {
  const char* what = "agpt_embed_fwd";
  if (T < 0 || V < 1 || D < 1) return invalid(what, "T < 0, V < 1 or D < 1");
  if (token_bits != 32 && token_bits != 64) return invalid(what, "token_bits must be 32 or 64");
  if (dtype != AGPT_DTYPE_F32 && dtype != AGPT_DTYPE_BF16) return invalid(what, "unknown dtype");
  if (T == 0) return AGPT_OK;
  if (!table || !tokens || !x) return invalid(what, "null pointer");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(table, es) || !aligned(x, es) || !aligned(tokens, token_bits / 8))
    return invalid(what, "a pointer is not aligned to its elements");
  const bool wide = static_cast<int64_t>(D) * es % 16 == 0 && aligned(table, 16) && aligned(x, 16);
  with_dtype(dtype, wide, [&](auto e, auto vc) {
    using E = decltype(e);
    constexpr int W = decltype(vc)::value;
    const int lanes = lanes_for(D, W), rpb = kThreads / lanes;
    const int64_t need = (T + rpb - 1) / rpb;
    const int gx = static_cast<int>(need < 8192 ? need : 8192);
    auto go = [&](auto tok) {
      using I = decltype(tok);
      hipLaunchKernelGGL((embed_fwd_kernel<E, I, W>), dim3(gx), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                         static_cast<const E*>(table), static_cast<const I*>(tokens), scale, static_cast<E*>(x), T, V,
                         D, lanes, gx);
    };
    if (token_bits == 32) go(int32_t{});
    else go(int64_t{});
  });
  return launch_status(what);
}

extern "C" int64_t agpt_embed_plan_ints(int64_t T, int64_t V) { return T < 0 || V < 1 ? 0 : 2 * T + V + 1; }

// Digit counts per tile, digit totals, and a second pair of keys and rows.
extern "C" int64_t agpt_embed_plan_workspace_bytes(int64_t T, int64_t V) {
  if (T < 0 || V < 1) return 0;
  return 4 * (kDigits * (tiles_of(T) + 1) + 2 * T);
}

extern "C" int agpt_embed_plan(const void* tokens, int token_bits, int64_t T, int64_t V, int32_t* plan,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "agpt_embed_plan";
  if (const int rc = check_counts(what, T, V)) return rc;
  if (token_bits != 32 && token_bits != 64) return invalid(what, "token_bits must be 32 or 64");
  if (!plan || (T > 0 && (!tokens || !workspace))) return invalid(what, "null pointer");
  if (!aligned(plan, 4) || !aligned(workspace, 4) || !aligned(tokens, token_bits / 8))
    return invalid(what, "a pointer is not aligned to its elements");
  if (workspace_bytes < agpt_embed_plan_workspace_bytes(T, V))
    return invalid(what, "workspace smaller than agpt_embed_plan_workspace_bytes");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  int32_t *order = plan, *keys = plan + T, *offsets = plan + 2 * T;
  int passes;
  const int bits = digit_bits(V, &passes), digits = 1 << bits;
  if (T > 0) {
    const int tiles = static_cast<int>(tiles_of(T));
    int32_t* counts = static_cast<int32_t*>(workspace);
    int32_t* totals = counts + static_cast<int64_t>(kDigits) * tiles;
    int32_t* keys2 = totals + kDigits;
    int32_t* rows2 = keys2 + T;
    const void* kin = tokens;
    const int32_t* rin = nullptr;
    for (int p = 0; p < passes; ++p) {
      const bool last_here = (passes - 1 - p) % 2 == 0;  // the last pass writes the plan
      int32_t *kout = last_here ? keys : keys2, *rout = last_here ? order : rows2;
      auto go = [&](auto tok, auto first) {
        using I = decltype(tok);
        constexpr bool kFirst = decltype(first)::value;
        const I* k = static_cast<const I*>(kin);
        hipLaunchKernelGGL((hist_kernel<I, kFirst>), dim3(tiles), dim3(kThreads), 0, st, k, T, V, p * bits, digits, counts,
                           tiles);
        hipLaunchKernelGGL(scan_kernel, dim3(digits), dim3(kThreads), 0, st, counts, tiles, totals);
        hipLaunchKernelGGL((place_kernel<I, kFirst>), dim3(tiles), dim3(kThreads), 0, st, k, rin, T, V, p * bits, bits,
                           counts, totals, tiles, kout, rout, passes == 1 ? offsets : static_cast<int32_t*>(nullptr));
      };
      if (p > 0) go(int32_t{}, std::false_type{});
      else if (token_bits == 32) go(int32_t{}, std::true_type{});
      else go(int64_t{}, std::true_type{});
      kin = kout;
      rin = rout;
    }
  }
  if (T == 0 || passes > 1)
    hipLaunchKernelGGL(offsets_kernel, dim3(static_cast<unsigned>(V / kThreads + 1)), dim3(kThreads), 0, st, keys,
                     static_cast<int32_t>(T), static_cast<int32_t>(V), offsets);
  return launch_status(what);
}

// Two partial rows per span.
extern "C" int64_t agpt_embed_bwd_workspace_floats(int64_t T, int D) {
  if (T < 0 || D < 1) return 0;
  const int R = span_rows(T);
  return 2 * ((T + R - 1) / R) * D;
}

extern "C" int agpt_embed_bwd(const void* dx, int64_t ld_dx, const int32_t* plan, float scale, float* d_table,
                              float* workspace, int64_t workspace_floats, int64_t T, int64_t V, int D, int dtype,
                              void* stream) {
  const char* what = "agpt_embed_bwd";
  if (const int rc = check_counts(what, T, V)) return rc;
  if (D < 1 || ld_dx < D) return invalid(what, "D < 1 or a row stride smaller than D");
  if (dtype != AGPT_DTYPE_F32 && dtype != AGPT_DTYPE_BF16) return invalid(what, "unknown dtype");
  if (!d_table || (T > 0 && (!dx || !plan || !workspace))) return invalid(what, "null pointer");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(dx, es) || !aligned(plan, 4) || !aligned(d_table, 4) || !aligned(workspace, 4))
    return invalid(what, "a pointer is not aligned to its elements");
  if (workspace_floats < agpt_embed_bwd_workspace_floats(T, D))
    return invalid(what, "workspace smaller than agpt_embed_bwd_workspace_floats");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (T == 0) {
    const int64_t need = (V * D + kThreads - 1) / kThreads;
    const int gx = static_cast<int>(need < 8192 ? need : 8192);
    hipLaunchKernelGGL(zero_kernel, dim3(gx), dim3(kThreads), 0, st, d_table, V * D, gx);
    return launch_status(what);
  }
  const int R = span_rows(T), spans = static_cast<int>((T + R - 1) / R);
  const int64_t waves = (V + kWaves - 1) / kWaves;
  if (waves + spans > 0x7fffffff) return invalid(what, "T and V too large together");
  const int32_t *order = plan, *keys = plan + T, *offsets = plan + 2 * T;
  const bool wide = wide_rows(D, ld_dx, es, dx, d_table);
  with_dtype(dtype, wide, [&](auto e, auto vc) {
    using E = decltype(e);
    constexpr int W = decltype(vc)::value;
    hipLaunchKernelGGL((sums_kernel<E, W>), dim3(static_cast<unsigned>(spans + waves)), dim3(kThreads), 0, st,
                       static_cast<const E*>(dx), ld_dx, order, keys, offsets, scale, d_table, workspace,
                       static_cast<int32_t>(T), static_cast<int32_t>(V), D, R, spans, lanes_for(D, W));
  });
  if (const int rc = launch_status(what)) return rc;
  int lanes = 1;
  while (lanes < D && lanes < 128) lanes *= 2;
  hipLaunchKernelGGL(join_kernel, dim3(spans), dim3(kJoin), 0, st, workspace, keys, offsets, scale, d_table,
                     static_cast<int32_t>(T), static_cast<int32_t>(V), D, R, lanes);
  return launch_status(what);
}

namespace {

// The one-launch form: log2 of its ranges, or -1 where sorting first is taken.
// Every workgroup reads all tokens, so it is for batches of at most kDirectRows
// rows, and for at most kDirectReads token reads in all.
constexpr int64_t kDirectRows = 16384, kDirectReads = int64_t{1} << 25;
int direct_ranges(int64_t T, int64_t V, int D, int width) {
  if (T < 1 || T > kDirectRows) return -1;
  const int64_t slices = (D + 64 * width - 1) / (64 * width);
  int lr = 0;
  while ((static_cast<int64_t>(kLocal) << lr) < V || ((slices << lr) < 512 && (int64_t{1} << lr) < V)) ++lr;
  return (slices << lr) * T <= kDirectReads ? lr : -1;
}

}  // namespace

// The plan, then the larger of what making it and summing by it need.
extern "C" int64_t agpt_embed_bwd_tokens_workspace_bytes(int64_t T, int64_t V, int D) {
  if (T < 0 || V < 1 || D < 1) return 0;
  const int64_t a = agpt_embed_plan_workspace_bytes(T, V), b = 4 * agpt_embed_bwd_workspace_floats(T, D);
  return 4 * agpt_embed_plan_ints(T, V) + (a > b ? a : b);
}

extern "C" int agpt_embed_bwd_tokens(const void* dx, int64_t ld_dx, const void* tokens, int token_bits, float scale,
                                     float* d_table, void* workspace, int64_t workspace_bytes, int64_t T, int64_t V, int D,
                                     int dtype, void* stream) {
  const char* what = "agpt_embed_bwd_tokens";
  if (const int rc = check_counts(what, T, V)) return rc;
  if (D < 1 || ld_dx < D) return invalid(what, "D < 1 or a row stride smaller than D");
  if (token_bits != 32 && token_bits != 64) return invalid(what, "token_bits must be 32 or 64");
  if (dtype != AGPT_DTYPE_F32 && dtype != AGPT_DTYPE_BF16) return invalid(what, "unknown dtype");
  if (!d_table || !workspace || (T > 0 && (!dx || !tokens))) return invalid(what, "null pointer");
  const int es = dtype == AGPT_DTYPE_F32 ? 4 : 2;
  if (!aligned(dx, es) || !aligned(tokens, token_bits / 8) || !aligned(d_table, 4) || !aligned(workspace, 4))
    return invalid(what, "a pointer is not aligned to its elements");
  if (workspace_bytes < agpt_embed_bwd_tokens_workspace_bytes(T, V, D))
    return invalid(what, "workspace smaller than agpt_embed_bwd_tokens_workspace_bytes");
  const bool wide = wide_rows(D, ld_dx, es, dx, d_table);
  const int width = !wide ? 1 : (dtype == AGPT_DTYPE_F32 ? 4 : 8);
  const int lr = direct_ranges(T, V, D, width);
  if (lr < 0) {
    int32_t* plan = static_cast<int32_t*>(workspace);
    int32_t* rest = plan + agpt_embed_plan_ints(T, V);
    const int64_t bytes = workspace_bytes - 4 * agpt_embed_plan_ints(T, V);
    if (const int rc = agpt_embed_plan(tokens, token_bits, T, V, plan, rest, bytes, stream)) return rc;
    return agpt_embed_bwd(dx, ld_dx, plan, scale, d_table, reinterpret_cast<float*>(rest), bytes / 4, T, V, D, dtype, stream);
  }
  with_dtype(dtype, wide, [&](auto e, auto vc) {
    using E = decltype(e);
    constexpr int W = decltype(vc)::value;
    int lanes = 1;
    while (lanes * W < D && lanes < 64) lanes *= 2;
    const dim3 grid(static_cast<unsigned>(((D + 64 * W - 1) / (64 * W)) << lr));
    auto go = [&](auto tok, auto cap) {
      using I = decltype(tok);
      hipLaunchKernelGGL((direct_kernel<E, I, W, decltype(cap)::value>), grid, dim3(kDirect), 0,
                         static_cast<hipStream_t>(stream), static_cast<const E*>(dx), ld_dx, static_cast<const I*>(tokens),
                         scale, d_table, static_cast<int>(T), V, D, lr, lanes);
    };
    auto size = [&](auto tok) {
      if (T <= 2048) go(tok, std::integral_constant<int, 2048>{});
      else go(tok, std::integral_constant<int, kDirectRows>{});
    };
    if (token_bits == 32) size(int32_t{});
    else size(int64_t{});
  });
  return launch_status(what);
}
