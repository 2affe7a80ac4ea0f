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
// Sums: a token of up to 16 rows is summed by one group of lanes that gathers
// them; a longer one by workgroups over spans of the sorted rows, and the pieces
// of one that goes over several spans are added in span order.
//
// HBM bounds the sums, launches and the waits of a short sort the rest: 2^20 rows of
// 128 fp32 over 65 tokens 105 us for the sums (545 MB at 5.2 TB/s) and 30 for order,
// offsets and pieces; 16K rows of 1024 bf16 over 50,000 tokens 64 (238 MB at 3.7) and
// 21. The lookup of 64K such rows takes 47 us (237 MB at 5.0).

#include "rows.h"
#include "../../include/agpt_embed.h"

#include <type_traits>

namespace {

using namespace agpt_rows;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxSpan = 512;

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
// Workgroups 0 .. spans - 1 take a span of sorted rows each. A token of up to
// kShort rows is summed by a group of lanes in the span where it begins. A longer
// one is summed by the whole workgroup, at once where it lies in one span, else in
// pieces to part[2 span] (begun in an earlier span) and part[2 span + 1] (begins
// here). The workgroups after them write the zeros of the tokens without rows, so
// that the gathers, a chain of waits each, start first: 16K rows over 50,000 tokens
// of 1024 bf16 from HBM took 84 us with a wave per token in token order, 64 in this
// one with a whole row to a lane group and spans of eight rows (a fill of dE and a
// copy of dx: 44).
constexpr int kShort = 16;
constexpr int kTokens = 4;   // of a lane group at a time, their first rows on their way together
constexpr int kZeroRows = 64;

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void sums_kernel(const T* __restrict__ dx, int64_t ld,
                                                        const int32_t* __restrict__ order,
                                                        const int32_t* __restrict__ keys,
                                                        const int32_t* __restrict__ offsets, float scale,
                                                        float* __restrict__ dE, float* __restrict__ part, int32_t n,
                                                        int32_t vocab, int D, int R, int spans, int lanes) {
  const int tid = thread_x(), blk = block_x();
  if (blk < spans) {
    __shared__ float red[kThreads * V];
    __shared__ int32_t many[kMaxSpan / kShort + 1], few_at[kMaxSpan], few_v[kMaxSpan], few_n[kMaxSpan];
    __shared__ int n_many, n_few;
    const int32_t s0 = blk * R, s1 = s0 + R < n ? s0 + R : n;
    if (tid == 0) n_many = n_few = 0;
    __syncthreads();
    // the span's tokens (listed in any order, each has a sum of its own): the short ones that begin in it, the
    // long ones that do and the one that it begins within
    for (int32_t p = s0 + tid; p < s1; p += kThreads) {
      const int32_t v = keys[p];
      if (v >= vocab) continue;
      const int32_t a = offsets[v];
      if (a != p && p != s0) continue;
      const int32_t count = offsets[v + 1] - a;
      if (count > kShort) {
        many[atomicAdd(&n_many, 1)] = v;
      } else if (a == p) {
        const int q = atomicAdd(&n_few, 1);
        few_at[q] = p;
        few_v[q] = v;
        few_n[q] = count;
      }
    }
    __syncthreads();
    const int slots = kThreads / lanes, slot = tid / lanes;
    for (int m = 0; m < n_many; ++m) {
      const int32_t v = many[m], a = offsets[v], b = offsets[v + 1];
      const int32_t p0 = a > s0 ? a : s0, p1 = b < s1 ? b : s1;
      const bool whole = a >= s0 && b <= s1;
      float* out = whole ? dE + static_cast<int64_t>(v) * D : part + (2 * static_cast<int64_t>(blk) + (a >= s0)) * D;
      for (int c0 = 0; c0 < D; c0 += lanes * V) {
        const int c = c0 + (tid & (lanes - 1)) * V;
        float s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = 0.0f;
        if (c < D) {
#pragma unroll 8
          for (int j = p0 + slot; j < p1; j += slots) {
            float x[V];
            load_row<V>(dx + order[j] * ld + c, x);
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += x[i];
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) red[tid * V + i] = s[i];
        __syncthreads();
        if (slot == 0 && c < D) {
          for (int q = 1; q < slots; ++q)
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += red[(q * lanes + tid) * V + i];
#pragma unroll
          for (int i = 0; i < V; ++i) out[c + i] = whole ? s[i] * scale : s[i];
        }
        __syncthreads();
      }
    }
    for (int q = slot * kTokens; q < n_few; q += slots * kTokens) {
      int32_t at[kTokens], count[kTokens], row[kTokens];
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        const bool in = q + k < n_few;
        at[k] = in ? few_at[q + k] : 0;
        count[k] = in ? few_n[q + k] : 0;
        row[k] = in ? order[at[k]] : 0;
      }
      for (int c = (tid & (lanes - 1)) * V; c < D; c += lanes * V) {
        float s[kTokens][V];
#pragma unroll
        for (int k = 0; k < kTokens; ++k)
          if (count[k] > 0) load_row<V>(dx + row[k] * ld + c, s[k]);
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
          if (count[k] == 0) continue;
#pragma unroll 8
          for (int j = 1; j < count[k]; ++j) {
            float x[V];
            load_row<V>(dx + order[at[k] + j] * ld + c, x);
#pragma unroll
            for (int i = 0; i < V; ++i) s[k][i] += x[i];
          }
#pragma unroll
          for (int i = 0; i < V; ++i) s[k][i] *= scale;
          store_row<V>(dE + static_cast<int64_t>(few_v[q + k]) * D + c, s[k]);
        }
      }
    }
    return;
  }
  __shared__ int32_t off[kZeroRows + 1];
  const int64_t v0 = static_cast<int64_t>(blk - spans) * kZeroRows;
  if (tid <= kZeroRows) off[tid] = offsets[v0 + tid < vocab ? v0 + tid : vocab];
  __syncthreads();
  float zero[V];
#pragma unroll
  for (int i = 0; i < V; ++i) zero[i] = 0.0f;
  const int rows = kThreads / lanes;
  for (int k = tid / lanes; k < kZeroRows && v0 + k < vocab; k += rows) {
    if (off[k + 1] > off[k]) continue;
    for (int c = (tid & (lanes - 1)) * V; c < D; c += lanes * V) store_row<V>(dE + (v0 + k) * D + c, zero);
  }
}

// The long tokens that begin in one of a workgroup's `each` spans and go on past
// it: their pieces, dealt to slots of `lanes` columns, the slots added in order.
constexpr int kJoin = 1024;
__global__ __launch_bounds__(kJoin) void join_kernel(const float* __restrict__ part, const int32_t* __restrict__ keys,
                                                     const int32_t* __restrict__ offsets, float scale,
                                                     float* __restrict__ dE, int32_t n, int32_t vocab, int D, int R,
                                                     int lanes, int spans, int each) {
  __shared__ float red[kJoin];
  __shared__ int32_t many[kJoin];
  __shared__ int n_many;
  const int tid = thread_x(), slots = kJoin / lanes, slot = tid / lanes;
  const int c = block_y() * lanes + (tid & (lanes - 1));
  for (int first = block_x() * each, last = first + each; first < last; first += kJoin) {
    if (tid == 0) n_many = 0;
    __syncthreads();
    const int span = first + tid;
    if (span < last && span < spans) {
      const int32_t s0 = span * R, s1 = s0 + R < n ? s0 + R : n, v = keys[s1 - 1];
      if (v < vocab) {
        const int32_t a = offsets[v], b = offsets[v + 1];
        if (b - a > kShort && a >= s0 && b > s1) many[atomicAdd(&n_many, 1)] = span;  // (in any order)
      }
    }
    __syncthreads();
    const int found = n_many;
    for (int m = 0; m < found; ++m) {
      const int s0 = many[m];
      const int32_t v = keys[s0 * R + R - 1], end = (offsets[v + 1] - 1) / R;
      float s = 0.0f;
      if (c < D) {
        if (slot == 0) s = part[(2 * static_cast<int64_t>(s0) + 1) * D + c];
#pragma unroll 8
        for (int q = s0 + 1 + slot; q <= end; q += slots) s += part[2 * static_cast<int64_t>(q) * D + c];
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
}

__global__ __launch_bounds__(kThreads) void zero_kernel(float* __restrict__ p, int64_t n, int gx) {
  for (int64_t i = static_cast<int64_t>(block_x()) * kThreads + thread_x(); i < n; i += static_cast<int64_t>(gx) * kThreads)
    p[i] = 0.0f;
}

// ---- plans of short batches in one launch -----------------------------------------
constexpr int kList = 512, kListWaves = kList / 64;
constexpr int kLocal = 256;  // tokens of a workgroup's share of the vocabulary, at most

// Lists the rows (n of them) whose token `mine` takes, in row order, each wave
// over its own part of the batch: found[first of the wave ...], the wave's count
// returned; `each` sees every key. Keys are the tokens, V for padding.
template <typename I, typename Mine, typename Each>
__device__ __forceinline__ int list_rows(const I* __restrict__ tokens, int n, int64_t vocab, uint16_t* found, int first,
                                         int last, Mine&& mine, Each&& each) {
  const int lane = thread_x() & 63;
  const uint64_t below = (1ull << lane) - 1;
  constexpr int kFlight = 16;  // token loads in flight
  int cnt = 0;
  for (int i = first; i < last; i += kFlight * 64) {
    I tok[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) tok[u] = i + u * 64 + lane < last ? tokens[i + u * 64 + lane] : I{0};
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const bool in = i + u * 64 + lane < last;
      const int32_t k = key_of(tok[u], vocab);
      each(in, k);
      const bool take = in && mine(k);
      const uint64_t m = __ballot(take);
      if (take) found[first + cnt + __popcll(m & below)] = static_cast<uint16_t>(i + u * 64 + lane);
      cnt += __popcll(m);
    }
  }
  return cnt;
}

// next[wave][local] from the counts of a wave's listed rows to the first place of
// its rows of that local token; start[local] the token's first place (and
// start[kLocal] the listed rows' number). `mark(local, rows)` per local token.
template <typename Mark>
__device__ __forceinline__ void list_places(int (*next)[kLocal], int* start, int* wsum, Mark&& mark) {
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6;
  __syncthreads();
  int tot = 0;
  if (tid < kLocal)
    for (int w = 0; w < kListWaves; ++w) tot += next[w][tid];
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
    mark(tid, tot);
    if (tid == kLocal - 1) start[kLocal] = inc;
    for (int w = 0; w < kListWaves; ++w) {
      const int c = next[w][tid];
      next[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
}

// The stable places of a wave's listed rows: place(row, local, at).
template <typename Local, typename Place>
__device__ __forceinline__ void list_sort(const uint16_t* found, int first, int cnt, int* next, Local&& local_of,
                                          Place&& place) {
  const int lane = thread_x() & 63;
  const uint64_t below = (1ull << lane) - 1;
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
    if (in) at = next[d] + rank;
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) next[d] = at + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (in) place(row, d, at);
  }
}

// A workgroup owns the keys lo .. lo + per - 1 (of 0 .. V). It reads every token
// from L2, counts those below lo, which is where its own begin, and lists and
// sorts its own: no workgroup waits for another.
constexpr int kShortRows = 32768;  // rows' numbers fit 16 bits
template <typename I, int kCap>
__global__ __launch_bounds__(kList) void short_plan_kernel(const I* __restrict__ tokens, int n, int64_t vocab, int per,
                                                           int32_t* __restrict__ order, int32_t* __restrict__ keys,
                                                           int32_t* __restrict__ offsets) {
  __shared__ uint16_t found[kCap + kList];
  __shared__ int next[kListWaves][kLocal];
  __shared__ int start[kLocal + 1];
  __shared__ int wsum[kListWaves], fewer[kListWaves];
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6;
  const int64_t lo = static_cast<int64_t>(block_x()) * per, hi = lo + per;
  const int share = (n + kList - 1) / kList * 64, first = wave * share;
  int under = 0;
  const int cnt = list_rows(
      tokens, n, vocab, found, first, first + share < n ? first + share : n,
      [&](int32_t k) { return k >= lo && k < hi; },
      [&](bool in, int32_t k) { under += __popcll(__ballot(in && k < lo)); });
  for (int i = lane; i < kLocal; i += 64) next[wave][i] = 0;
  if (lane == 0) fewer[wave] = under;
  __builtin_amdgcn_wave_barrier();
  auto local_of = [&](int row) { return static_cast<int>(key_of(tokens[row], vocab) - lo); };
  for (int j = lane; j < cnt; j += 64) atomicAdd(&next[wave][local_of(found[first + j])], 1);
  list_places(next, start, wsum, [](int, int) {});
  int base = 0;
  for (int w = 0; w < kListWaves; ++w) base += fewer[w];
  if (tid < per && lo + tid <= vocab) offsets[lo + tid] = base + start[tid];
  list_sort(found, first, cnt, next[wave], local_of, [&](int row, int d, int at) {
    order[base + at] = row;
    keys[base + at] = static_cast<int32_t>(lo) + d;
  });
}

// ---- one launch for the shortest batches ----------------------------------------------
// A workgroup owns the tokens v = range (mod ranges), ranges a power of two (so
// that neighbouring, often equally frequent ids part), and `lanes` V columns. It
// reads every token of the batch from L2, lists the rows of its own, sorts the
// list (stable, by the token's number within the range: at most 256, one digit)
// and sums each token's rows, `lanes` lanes per token; a token of many rows takes
// all of the workgroup's lane groups. Few columns to a workgroup spread such a
// token over more CUs, at the price of reading the tokens more often.
constexpr int kDirectRows = 2048;  // of a batch at most

template <typename T, typename I, int V>
__global__ __launch_bounds__(kList) void direct_kernel(const T* __restrict__ dx, int64_t ld,
                                                       const I* __restrict__ tokens, float scale,
                                                       float* __restrict__ dE, int n, int64_t vocab, int D, int log_ranges,
                                                       int lanes) {
  __shared__ uint16_t found[kDirectRows + kList], rows[kDirectRows + kList];
  __shared__ int next[kListWaves][kLocal];
  __shared__ int start[kLocal + 1], many[kLocal], n_many;
  __shared__ int wsum[kListWaves];
  __shared__ float red[kList * V];
  constexpr int kLong = 32;  // rows that a lane group sums by itself
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6, blk = block_x();
  const int ranges = 1 << log_ranges, range = blk & (ranges - 1), slice = blk >> log_ranges;
  const int per_range = static_cast<int>((vocab + ranges - 1) >> log_ranges);
  const int share = (n + kList - 1) / kList * 64, first = wave * share;
  const int cnt = list_rows(
      tokens, n, vocab, found, first, first + share < n ? first + share : n,
      [&](int32_t k) { return k < vocab && (k & (ranges - 1)) == range; }, [](bool, int32_t) {});
  for (int i = lane; i < kLocal; i += 64) next[wave][i] = 0;
  if (tid == 0) n_many = 0;
  __builtin_amdgcn_wave_barrier();
  auto local_of = [&](int row) { return static_cast<int>(static_cast<int64_t>(tokens[row]) >> log_ranges); };
  for (int j = lane; j < cnt; j += 64) atomicAdd(&next[wave][local_of(found[first + j])], 1);
  list_places(next, start, wsum, [&](int k, int count) {
    if (count > kLong) many[atomicAdd(&n_many, 1)] = k;  // (in any order: each token has a sum of its own)
  });
  list_sort(found, first, cnt, next[wave], local_of, [&](int row, int, int at) { rows[at] = static_cast<uint16_t>(row); });
  __syncthreads();

  const int groups = kList / lanes, grp = tid / lanes, c = (slice * lanes + (tid & (lanes - 1))) * V;
  auto sum_rows = [&](int a, int b, int step, float (&s)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.0f;
#pragma unroll 8
    for (int j = a; j < b; j += step) {
      float x[V];
      load_row<V>(dx + rows[j] * ld + c, x);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += x[i];
    }
  };
  // the tokens of many rows, one after the other: rows dealt to the groups, the groups' sums added in order
  for (int m = 0; m < n_many; ++m) {
    const int k = many[m], a = start[k], b = start[k + 1];
    const int64_t v = (static_cast<int64_t>(k) << log_ranges) | range;
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.0f;
    if (c < D) sum_rows(a + grp, b, groups, s);
#pragma unroll
    for (int i = 0; i < V; ++i) red[tid * V + i] = s[i];
    __syncthreads();
    // by halves: 64 lanes' worth of groups and more fold in log2(groups) steps
    for (int o = groups / 2; o > 0; o /= 2) {
      if (grp < o) {
#pragma unroll
        for (int i = 0; i < V; ++i) red[tid * V + i] += red[(tid + o * lanes) * V + i];
      }
      __syncthreads();
    }
    if (grp == 0 && c < D) {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = red[tid * V + i] * scale;
      store_row<V>(dE + v * D + c, s);
    }
    __syncthreads();
  }
  if (c >= D) return;
  for (int k = grp; k < per_range; k += groups) {
    const int64_t v = (static_cast<int64_t>(k) << log_ranges) | range;
    const int a = start[k], b = start[k + 1];
    if (v >= vocab || b - a > kLong) continue;
    float s[V];
    sum_rows(a, b, 1, s);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= scale;
    store_row<V>(dE + v * D + c, s);
  }
}

constexpr int kMaxWidth = 1 << 30;  // columns and steps past the last one stay in 32 bits
constexpr int64_t kMaxCount = 0x7fffffff - 4096;  // places and steps past the last one stay in 32 bits

int digit_bits(int64_t V, int* passes) {
  int bits = 1;
  while ((V >> bits) != 0) ++bits;  // keys 0 .. V
  *passes = (bits + kMaxBits - 1) / kMaxBits;
  return (bits + *passes - 1) / *passes;
}

// Keys of a workgroup where a plan is made in one launch, 0 where it is sorted:
// every workgroup reads all tokens, so it is for at most kShortRows rows (half of
// them where the sort is a single pass) and kShortReads token reads in all. Plan
// and sums of rows of 128, one launch against sorting: 32K rows over 300 tokens
// 39 and 50 us, over 50,000 59 and 60, over 65 36 and 28; 16K rows over 65 25 and 27.
constexpr int64_t kShortReads = int64_t{1} << 25;
int short_plan_keys(int64_t T, int64_t V) {
  if (T > (V < kDigits ? kShortRows / 2 : kShortRows)) return 0;
  const int64_t per = V / 256 + 1 < kLocal ? V / 256 + 1 : kLocal;
  return (V / per + 1) * T <= kShortReads ? static_cast<int>(per) : 0;
}

// Rows of a span: enough spans to fill the chip, few enough pieces to add.
int span_rows(int64_t T) {
  int R = 8;
  while (R < kMaxSpan && T / R > 2048) R *= 2;
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
  if (D > kMaxWidth) return invalid(what, "D must be at most 2^30");
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
  if (const int per = short_plan_keys(T, V)) {
    const dim3 grid(static_cast<unsigned>(V / per + 1));
    auto go = [&](auto tok, auto cap) {
      using I = decltype(tok);
      hipLaunchKernelGGL((short_plan_kernel<I, decltype(cap)::value>), grid, dim3(kList), 0, st,
                         static_cast<const I*>(tokens), static_cast<int>(T), V, per, order, keys, offsets);
    };
    auto size = [&](auto tok) {  // (the smaller list leaves a CU room for three workgroups)
      if (T <= 16384) go(tok, std::integral_constant<int, 16384>{});
      else go(tok, std::integral_constant<int, kShortRows>{});
    };
    if (token_bits == 32) size(int32_t{});
    else size(int64_t{});
    return launch_status(what);
  }
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
  if (D > kMaxWidth) return invalid(what, "D must be at most 2^30");
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
  const int32_t *order = plan, *keys = plan + T, *offsets = plan + 2 * T;
  const bool wide = wide_rows(D, ld_dx, es, dx, d_table);
  with_dtype(dtype, wide, [&](auto e, auto vc) {
    using E = decltype(e);
    constexpr int W = decltype(vc)::value;
    const int lanes = lanes_for(D, W);
    const int64_t blocks = spans + (V + kZeroRows - 1) / kZeroRows;  // far below 2^31
    hipLaunchKernelGGL((sums_kernel<E, W>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st,
                       static_cast<const E*>(dx), ld_dx, order, keys, offsets, scale, d_table, workspace,
                       static_cast<int32_t>(T), static_cast<int32_t>(V), D, R, spans, lanes);
  });
  if (const int rc = launch_status(what)) return rc;
  if (spans == 1) return AGPT_OK;  // no token goes over spans
  int lanes = 1;
  while (lanes < D && lanes < 128) lanes *= 2;
  const int each = (spans + 255) / 256;
  hipLaunchKernelGGL(join_kernel, dim3((spans + each - 1) / each, (D + lanes - 1) / lanes), dim3(kJoin), 0, st, workspace,
                     keys, offsets, scale, d_table, static_cast<int32_t>(T), static_cast<int32_t>(V), D, R, lanes, spans,
                     each);
  return launch_status(what);
}

namespace {

// The one-launch form: log2 of its ranges, or -1 where a plan is made first.
// Every workgroup reads all tokens, and one long token's rows are one workgroup's:
// for at most kDirectRows rows and kShortReads token reads in all.
int direct_ranges(int64_t T, int64_t V, int D, int width, int* lanes) {
  if (T < 1 || T > kDirectRows) return -1;
  for (*lanes = 16; *lanes <= 64; *lanes *= 2) {  // the fewest columns that the reads allow
    const int64_t slices = (D + *lanes * width - 1) / (*lanes * width);
    int lr = 0;
    while ((static_cast<int64_t>(kLocal) << lr) < V || ((slices << lr) < 512 && (int64_t{1} << lr) < V)) ++lr;
    if ((slices << lr) * T <= kShortReads) return lr;
  }
  return -1;
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
  if (D > kMaxWidth) return invalid(what, "D must be at most 2^30");
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
  int lanes;
  const int lr = direct_ranges(T, V, D, width, &lanes);
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
    const dim3 grid(static_cast<unsigned>(((D + lanes * W - 1) / (lanes * W)) << lr));
    auto go = [&](auto tok) {
      using I = decltype(tok);
      hipLaunchKernelGGL((direct_kernel<E, I, W>), grid, dim3(kList), 0, static_cast<hipStream_t>(stream),
                         static_cast<const E*>(dx), ld_dx, static_cast<const I*>(tokens), scale, d_table,
                         static_cast<int>(T), V, D, lr, lanes);
    };
    if (token_bits == 32) go(int32_t{});
    else go(int64_t{});
  });
  return launch_status(what);
}
