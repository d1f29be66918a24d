// Embedding lookup with scaling and pooling, and its gradient by sorted ids,
// for MI355X (gfx950, CDNA4).
//
//   out[b]    = T(c[b] * sum over l of w[b,l] * table[ids[b,l]])
//   dw[b,l]   = c[b] * <table[ids[b,l]], dy[b]>
//   dtable[v] = T(sum over (b,l) with ids[b,l] = v of c[b] * w[b,l] * dy[b])
//
// with c[b] = scale / norm, norm 1, n or sqrt(n) for n ids in bag b. Ids
// below zero are no tokens; ids past the table make their output NaN and
// have no gradient. Sums are in 32 bits, in an order that the inputs alone
// decide: no atomic adds to a sum.
//
// All of it moves rows, so it is bound by memory, or by launches where there
// are few tokens.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "embedding_kernels.h"

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

namespace {

constexpr uint32_t kNone = 0xffffffffu;

__device__ inline float as_f32(float v) { return v; }
__device__ inline float as_f32(__bf16 v) { return (float)v; }
__device__ inline float as_f32(_Float16 v) { return (float)v; }

__device__ inline float load_any(const void* p, int64_t i, int type) {
  if (type == EDL_T_F32) return static_cast<const float*>(p)[i];
  if (type == EDL_T_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}

template <typename T, int N>
struct Vec {
  typedef T type __attribute__((ext_vector_type(N)));
  type v;
  __device__ float get(int i) const { return as_f32(v[i]); }
  __device__ void set(int i, float x) { v[i] = (T)x; }
};
template <typename T>
struct Vec<T, 1> {
  T v;
  __device__ float get(int) const { return as_f32(v); }
  __device__ void set(int, float x) { v = (T)x; }
};

__device__ inline int64_t load_id(const void* ids, bool wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i]
              : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// U neighbours at `at`, of which n are there: wide loads where all are, as a
// load costs its instruction for every row of lanes, not its bytes
template <typename T, int U, int ALIGN>
__device__ inline void load_run(const void* p, int64_t at, T* to) {
  constexpr int W = 16 / sizeof(T) < U ? 16 / sizeof(T) : U;
  typedef T vec __attribute__((ext_vector_type(W), aligned(ALIGN)));
#pragma unroll
  for (int u = 0; u < U; u += W) {
    const vec v = *reinterpret_cast<const vec*>(static_cast<const T*>(p) + at + u);
#pragma unroll
    for (int q = 0; q < W; ++q) to[u + q] = v[q];
  }
}
template <int U>
__device__ inline void load_ids(const void* ids, bool wide, int64_t at, int n,
                                int64_t* id) {
  if (n < U) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = u < n ? load_id(ids, wide, at + u) : -1;
  } else if (wide) {
    load_run<int64_t, U, 8>(ids, at, id);
  } else {
    int32_t v[U];
    load_run<int32_t, U, 4>(ids, at, v);
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = v[u];
  }
}
template <int U>
__device__ inline void load_weights(const void* p, int type, int64_t at, int n,
                                    float* w) {
  if (p == nullptr) {
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = 1.f;
  } else if (type == EDL_T_F32 && n >= U) {
    load_run<float, U, 4>(p, at, w);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = u < n ? load_any(p, at + u, type) : 0.f;
  }
}

// lanes that share a row: a power of two, at most a wave
__host__ __device__ inline int lanes_of(int D, int vec) {
  int n = (D + vec - 1) / vec, l = 1;
  while (l < n && l < 64) l <<= 1;
  return l;
}
// a row's pieces of lanes_of() loads
__host__ __device__ inline int pieces_of(int D, int vec) {
  const int each = lanes_of(D, vec) * vec;
  return (D + each - 1) / each;
}

// --------------------------------- lookup ---------------------------------
// A row is read by the few lanes that its width takes, 8 ids at a time so
// that 8 rows are in flight; `subs` such groups share a bag, each taking
// every so-many-th eight, where bags alone are too few to fill the chip.
// Bound by random rows: 16384 bags of up to 50 rows of 128 bytes 15.6 us, 3.0
// TB/s with the padding's ids.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void lookup_kernel(edl_bag a, int subs,
                                                     int64_t block0) {
  typedef Vec<T, VEC> V;
  constexpr int U = 8;
  const int lanes = lanes_of(a.D, VEC), pieces = pieces_of(a.D, VEC);
  const int lane = threadIdx.x & 63;
  const int sub = (lane / lanes) & (subs - 1);
  const int64_t unit =
      ((block0 + blockIdx.x) * 256 + threadIdx.x) / (lanes * subs);
  const int64_t bag = unit / pieces;
  const int col = ((int)(unit % pieces) * lanes + (lane & (lanes - 1))) * VEC;
  if (bag >= a.B) return;  // whole groups of lanes * subs
  const bool mine = col < a.D;
  const int at = mine ? col : 0;
  const T* table = static_cast<const T*>(a.table) + at;

  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  int count = 0;
  for (int l0 = sub * U; l0 < a.L; l0 += subs * U) {
    int64_t id[U];
    load_ids<U>(a.ids, a.ids64, bag * a.L + l0, a.L - l0, id);
    bool any = false;
#pragma unroll
    for (int u = 0; u < U; ++u) any |= id[u] >= 0;
    if (!__any(any)) continue;  // behind the ends of short bags
    float weight[U];
    load_weights<U>(a.weights, a.w_type, bag * a.L + l0, a.L - l0, weight);
    V row[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      row[u].v = *reinterpret_cast<const decltype(row[u].v)*>(
          table + ((uint64_t)id[u] < (uint64_t)a.V ? id[u] : 0) * a.ld);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] < 0) continue;
      ++count;
      const float w = weight[u];
      const float bad = id[u] < a.V ? 0.f : __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        acc[k] += bad == 0.f ? w * row[u].get(k) : bad;
    }
  }
  for (int o = lanes; o < lanes * subs; o <<= 1) {
    count += __shfl_xor(count, o);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor(acc[k], o);
  }
  if (sub != 0) return;
  const float n = (float)(count > 1 ? count : 1);
  float c = a.scale;
  if (a.combiner == EDL_BAG_MEAN) c = a.scale / n;
  if (a.combiner == EDL_BAG_SQRTN) c = a.scale / sqrtf(n);
  if (a.coef && col == 0) a.coef[bag] = c;
  if (!mine) return;
  V o;
#pragma unroll
  for (int k = 0; k < VEC; ++k) o.set(k, acc[k] * c);
  *reinterpret_cast<decltype(o.v)*>(static_cast<T*>(a.out) + bag * a.D + col) =
      o.v;
}

// the weights' gradient: a group of lanes goes over a bag's ids, which lie
// in its lanes' registers four at a time (16384 bags of up to 50 ids, 64
// columns of bf16 19 us; eight at a time 24)
template <typename T, int VEC>
__global__ __launch_bounds__(256) void weight_grad_kernel(edl_bag a,
                                                          int64_t block0) {
  typedef Vec<T, VEC> V;
  constexpr int U = 4;
  const int lanes = lanes_of(a.D, VEC);
  const int64_t unit = ((block0 + blockIdx.x) * 256 + threadIdx.x) / lanes;
  const int l_lane = threadIdx.x & (lanes - 1);
  // eight ids of a bag to a unit, so that long bags spread
  const int eights = (a.L + 7) / 8;
  const int64_t bag = unit / eights;
  const int l0 = (int)(unit % eights) * 8;
  if (bag >= a.B) return;
  const T* dy = static_cast<const T*>(a.dy) + bag * a.D;
  const T* table = static_cast<const T*>(a.table);
  const float c = a.coef[bag];
  for (int l = l0; l < l0 + 8 && l < a.L; l += U) {
    int64_t id[U];
    float dot[U];
    load_ids<U>(a.ids, a.ids64, bag * a.L + l, a.L - l, id);
#pragma unroll
    for (int u = 0; u < U; ++u) dot[u] = 0.f;
    bool any = false;  // not behind the end of a short bag
#pragma unroll
    for (int u = 0; u < U; ++u) any |= id[u] >= 0;
    for (int col = l_lane * VEC; any && col < a.D; col += lanes * VEC) {
      V g, row[U];
      g.v = *reinterpret_cast<const decltype(g.v)*>(dy + col);
#pragma unroll
      for (int u = 0; u < U; ++u)
        row[u].v = *reinterpret_cast<const decltype(row[u].v)*>(
            table + ((uint64_t)id[u] < (uint64_t)a.V ? id[u] : 0) * a.ld +
            col);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dot[u] += row[u].get(k) * g.get(k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      for (int o = 1; o < lanes; o <<= 1) dot[u] += __shfl_xor(dot[u], o);
      if (l_lane == 0 && l + u < a.L)
        a.dw[bag * a.L + l + u] =
            (uint64_t)id[u] < (uint64_t)a.V ? dot[u] * c : 0.f;
    }
  }
}

// ---------------------------------- sort ----------------------------------
// Least significant digit first, stable, 9 or 11 bits a pass. A pass counts
// each tile's digits, adds the counts up by digit, and moves each tile's
// items: ranked by the wave (ballots find equal digits), brought in order in
// LDS, and written in runs. The first pass makes the keys from the ids.
struct Keys32 {  // an id of a table of V rows; V where it has none
  typedef uint32_t K;
  const void* ids;
  bool wide;
  int64_t V;
  __device__ K operator()(int64_t i) const {
    const int64_t v = load_id(ids, wide, i);
    return (uint64_t)v < (uint64_t)V ? (K)v : (K)V;
  }
};
struct Keys32Of {  // an id's low 32 bits
  typedef uint32_t K;
  const int64_t* ids;
  __device__ K operator()(int64_t i) const { return (K)ids[i]; }
};
struct Keys64 {  // any id; the sign bit turned, so that the order is theirs
  typedef uint64_t K;
  const int64_t* ids;
  __device__ K operator()(int64_t i) const {
    return (uint64_t)ids[i] ^ 0x8000000000000000ull;
  }
};
template <typename K_>
struct KeysOf {  // what the pass before wrote
  typedef K_ K;
  const K* keys;
  __device__ K operator()(int64_t i) const { return keys[i]; }
};

struct Plan4x11 {  // tiles of 256 * ITEMS, digits of up to BITS
  static constexpr int ITEMS = 4, BITS = 11;
};
struct Plan4x9 {
  static constexpr int ITEMS = 4, BITS = 9;
};
struct Plan16x9 {
  static constexpr int ITEMS = 16, BITS = 9;
};

// the lanes among `in` whose digit of BITS bits is this lane's
template <int BITS>
__device__ inline uint64_t same_digit(uint32_t d, bool in) {
  const uint64_t all = __ballot(in);
  uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const uint32_t mine = (uint32_t)((int32_t)(d << (31 - b)) >> 31);
    const uint64_t set = __ballot((int32_t)mine < 0);
    lo &= ~((uint32_t)set ^ mine);
    hi &= ~((uint32_t)(set >> 32) ^ mine);
  }
  return (uint64_t)hi << 32 | lo;
}
// a lane's rank among the wave's items of its digit so far, which `count`
// holds by digit: read by all, then moved on by the first of each digit
template <int BITS, typename C>
__device__ inline uint32_t rank_digit(volatile C* count, uint32_t d, bool in) {
  const uint64_t same = same_digit<BITS>(d, in);
  const uint32_t lower = __builtin_amdgcn_mbcnt_hi(
      (uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
  const uint32_t old = count[d];
  __builtin_amdgcn_wave_barrier();
  if (in && lower == 0) count[d] = (C)(old + __popcll(same));
  __builtin_amdgcn_wave_barrier();
  return old + lower;
}

// Zeros, by workgroups beside those of a sort, whose waits they fill, and past
// L2, which the sort uses: a whole gradient of 128 MB 144 us, 152 with all of
// them beside its first kernel, 158 with a launch of their own.
struct Zeros {
  uint8_t* to;  // on a border of 16 bytes
  int64_t bytes;
};
constexpr int kZeroBlocks = 1024;
template <int THREADS>
__device__ inline void fill_zeros(const Zeros& z, int64_t block,
                                  int64_t blocks) {
  const int64_t n = z.bytes / 16, step = blocks * THREADS;
  const u32x4 none = {0, 0, 0, 0};
  for (int64_t i = block * THREADS + threadIdx.x; i < n; i += step)
    __builtin_nontemporal_store(none, reinterpret_cast<u32x4*>(z.to) + i);
  if (block == 0 && threadIdx.x < z.bytes % 16)
    z.to[n * 16 + threadIdx.x] = 0;
}

// Workgroups go to the 8 XCDs in turn; this gives each XCD a run of
// neighbouring tiles. A digit's items from them, and their counts, lie
// together where they go, so that its L2 writes whole lines (a pass over 2.6
// million items 30 us, 35 in the order of launch).
__device__ inline int xcd_order(int bid, int n) {
  if (n < 8) return bid;
  const int xcd = bid & 7, idx = bid >> 3, q = n >> 3, r = n & 7;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

template <typename S, typename P>
__global__ __launch_bounds__(256) void sort_count_kernel(S src, int64_t N,
                                                         int shift, int bits,
                                                         int tiles,
                                                         uint32_t* counts,
                                                         Zeros zeros) {
  constexpr int ITEMS = P::ITEMS;
  if ((int)blockIdx.x >= tiles)
    return fill_zeros<256>(zeros, blockIdx.x - tiles, gridDim.x - tiles);
  __shared__ uint32_t h[1 << P::BITS];
  const int bins = 1 << bits;
  for (int d = threadIdx.x; d < bins; d += 256) h[d] = 0;
  __syncthreads();
  const int tile = xcd_order(blockIdx.x, tiles);
  const int64_t base = (int64_t)tile * (ITEMS * 256);
  if (base + ITEMS * 256 <= N) {  // four neighbours to a load
    typename S::K key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      key[k] = src(base + (k / 4 * 256 + threadIdx.x) * 4 + k % 4);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      atomicAdd(&h[(uint32_t)(key[k] >> shift) & (bins - 1)], 1u);
  } else {
    for (int64_t i = base + threadIdx.x; i < N; i += 256)
      atomicAdd(&h[(uint32_t)(src(i) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += 256)
    counts[(int64_t)d * tiles + tile] = h[d];
}

// exclusive sum over the 256 threads, and the total
__device__ inline uint32_t block_scan(uint32_t v, uint32_t* s4,
                                      uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t x = v;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) s4[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before += s4[w];
    all += s4[w];
  }
  __syncthreads();
  *total = all;
  return before + x - v;
}

// one digit's counts to offsets within the digit, and its total
__global__ __launch_bounds__(256) void sort_offsets_kernel(uint32_t* counts,
                                                           int tiles,
                                                           uint32_t* totals) {
  __shared__ uint32_t s4[4];
  uint32_t* row = counts + (int64_t)blockIdx.x * tiles;
  uint32_t run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + threadIdx.x;
    const uint32_t v = t < tiles ? row[t] : 0;
    uint32_t all;
    const uint32_t x = block_scan(v, s4, &all);
    if (t < tiles) row[t] = run + x;
    run += all;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

template <typename S, bool FIRST, typename P>
__global__ __launch_bounds__(256) void sort_move_kernel(
    S src, const uint32_t* __restrict__ pos_in, int64_t N, int shift, int bits,
    int tiles, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, typename S::K* __restrict__ keys_out,
    uint32_t* __restrict__ pos_out, Zeros zeros) {
  typedef typename S::K K;
  constexpr int ITEMS = P::ITEMS, kTile = ITEMS * 256, kBins = 1 << P::BITS;
  constexpr int kOwn = kBins / 256;  // neighbouring digits to a thread
  __shared__ K s_key[kTile];
  __shared__ uint32_t s_pos[kTile];
  __shared__ __align__(16) uint16_t cnt[4][kBins];  // a wave's, up to 1024
  __shared__ uint16_t local[kBins];  // a digit's first place in the tile
  __shared__ uint32_t goal[kBins];   // where it goes, less that place
  __shared__ uint32_t s4[4];
  if ((int)blockIdx.x >= tiles)
    return fill_zeros<256>(zeros, blockIdx.x - tiles, gridDim.x - tiles);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bins = 1 << bits;
  const int tile = xcd_order(blockIdx.x, tiles);
  const int64_t base = (int64_t)tile * kTile;
  const int64_t first = base + wave * (kTile / 4) + lane;
  K key[ITEMS];
  uint32_t pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t i = first + k * 64;
    const bool in = i < N;
    key[k] = in ? src(i) : 0;
    pos[k] = in ? (FIRST ? (uint32_t)i : pos_in[i]) : 0;
  }
  uint32_t tot[kOwn], at_tile[kOwn];
#pragma unroll
  for (int q = 0; q < kOwn; ++q) {
    const int d = tid * kOwn + q;
    tot[q] = d < bins ? totals[d] : 0;
    at_tile[q] = d < bins ? counts[(int64_t)d * tiles + tile] : 0;
  }
  for (int d = tid; d < 2 * kBins; d += 256)
    reinterpret_cast<uint32_t*>(&cnt[0][0])[d] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)
    rank[k] = rank_digit<P::BITS, uint16_t>(
        cnt[wave], (uint32_t)(key[k] >> shift) & (bins - 1),
        first + k * 64 < N);
  __syncthreads();
  uint32_t sum[kOwn], sums = 0, tots = 0;
#pragma unroll
  for (int q = 0; q < kOwn; ++q) {
    const int d = tid * kOwn + q;
    uint32_t s = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t t = cnt[w][d];
      cnt[w][d] = (uint16_t)s;
      s += t;
    }
    sum[q] = s;
    sums += s;
    tots += tot[q];
  }
  uint32_t all;
  uint32_t l0 = block_scan(sums, s4, &all);
  uint32_t g0 = block_scan(tots, s4, &all);
#pragma unroll
  for (int q = 0; q < kOwn; ++q) {
    const int d = tid * kOwn + q;
    local[d] = (uint16_t)l0;
    goal[d] = g0 + at_tile[q] - l0;
    l0 += sum[q];
    g0 += tot[q];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    if (first + k * 64 < N) {
      const uint32_t d = (uint32_t)(key[k] >> shift) & (bins - 1);
      const uint32_t at = local[d] + cnt[wave][d] + rank[k];
      s_key[at] = key[k];
      s_pos[at] = pos[k];
    }
  }
  __syncthreads();
  const int n = (int)(N - base < kTile ? N - base : kTile);
  for (int at = tid; at < n; at += 256) {
    const K key = s_key[at];
    const uint32_t to =
        goal[(uint32_t)(key >> shift) & (bins - 1)] + (uint32_t)at;
    keys_out[to] = key;
    pos_out[to] = s_pos[at];
  }
}

// Up to EDL_SORT_SMALL items: an item's place is how many come before it, by
// key and then by position, and it is counted. That is N^2 comparisons, but
// two instructions each and all of the chip's at once, where a sort in one
// workgroup waits for itself (6656 ids of 21 bits: 24 us in passes of 8 bits,
// 12 us counted and 4 for the runs). Sums of 8192 rows by id take 36 us so
// and 69 by the radix sort; of 16384, whose keys would take 128 KB of LDS, 62
// and 68. A workgroup has 32 items, and two lanes
// of each wave for each share those that they are compared with.
//
// IDS: ids of any value, less 2^31 below the first, which goes to info[0];
// info[1]: some lie too far from it for 32 bits, and all are compared in 64
// (8192 ids in 15 us, 13.5 in 32 bits; the whole call 48 us and 38, and 144
// where they went to the radix sort). The difference wraps at 2^64, so that
// ids at one end of int64 look near to the other's: their order and the keys'
// disagree, which is too far as well.
// Else rows of a table.
constexpr int kSmallThreads = 1024;
constexpr int kSmallItems = EDL_SORT_SMALL / kSmallThreads;
constexpr int kSmallWaves = kSmallThreads / 64;
constexpr int kSmallTile = 32, kSmallShares = kSmallThreads / kSmallTile;

// how many keys of places j0 to j1 come before the one at `place`
template <typename K, int kTile = kSmallTile>
__device__ inline uint32_t rank_among(const K* s_key, int place, int j0,
                                      int j1) {
  typedef K k4 __attribute__((ext_vector_type(4), aligned(16)));
  const int tile0 = place / kTile * kTile, tile1 = tile0 + kTile;
  const K key = s_key[place];
  uint32_t rank = 0;
  const auto four = [&](int j) {
    return *reinterpret_cast<const k4*>(s_key + j);
  };
#pragma unroll 4
  for (int j = j0; j < min(j1, tile0); j += 4) {  // equal ones come before
    const k4 o = four(j);
#pragma unroll
    for (int q = 0; q < 4; ++q) rank += o[q] <= key;
  }
  for (int j = max(j0, tile0); j < min(j1, tile1); j += 4) {
    const k4 o = four(j);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      rank += o[q] < key || (o[q] == key && j + q < place);
  }
#pragma unroll 4
  for (int j = max(j0, tile1); j < j1; j += 4) {  // and behind
    const k4 o = four(j);
#pragma unroll
    for (int q = 0; q < 4; ++q) rank += o[q] < key;
  }
  return rank;
}

template <typename S, bool IDS>
__global__ __launch_bounds__(kSmallThreads) void rank_small_kernel(
    S src, int N, uint32_t* keys_out, uint32_t* pos_out, int64_t* info,
    int tiles, Zeros zeros) {
  __shared__ __align__(16) uint64_t s_room[EDL_SORT_SMALL / (IDS ? 1 : 2)];
  __shared__ uint32_t s_rank[kSmallShares][kSmallTile];
  uint32_t* s_key = reinterpret_cast<uint32_t*>(s_room);
  if ((int)blockIdx.x >= tiles)
    return fill_zeros<kSmallThreads>(zeros, blockIdx.x - tiles,
                                     gridDim.x - tiles);
  const int tid = threadIdx.x;
  const int all = (N + 4 * kSmallShares - 1) / (4 * kSmallShares) *
                  (4 * kSmallShares);
  bool far = false;
  if constexpr (IDS) {
    const int64_t first = src.ids[0];
    const uint64_t low = (uint64_t)first - 0x80000000ull;
    uint32_t off = 0;
#pragma unroll
    for (int k = 0; k < kSmallItems; ++k) {
      const int i = k * kSmallThreads + tid;
      const int64_t id = src.ids[i < N ? i : 0];
      const uint64_t rel = (uint64_t)id - low;
      off |= (uint32_t)(rel >> 32) | ((id < first) != (rel < 0x80000000ull));
      if (i < all) s_key[i] = i < N ? (uint32_t)rel : kNone;
    }
    far = __syncthreads_or(off != 0);  // all alike
    if (blockIdx.x == 0 && tid == 0) {
      info[0] = (int64_t)low;
      info[1] = far;
    }
    if (far) {
#pragma unroll
      for (int k = 0; k < kSmallItems; ++k) {
        const int i = k * kSmallThreads + tid;
        if (i < all)
          s_room[i] = i < N ? (uint64_t)src.ids[i] ^ 0x8000000000000000ull
                            : ~0ull;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kSmallItems; ++k) {
      const int i = k * kSmallThreads + tid;
      if (i < all) s_key[i] = i < N ? (uint32_t)src(i) : kNone;
    }
  }
  __syncthreads();
  const int item = tid & (kSmallTile - 1), which = tid / kSmallTile;
  const int place = (int)blockIdx.x * kSmallTile + item;
  const int share = all / kSmallShares, j0 = which * share, j1 = j0 + share;
  uint32_t rank = far ? rank_among(s_room, place, j0, j1)
                      : rank_among(s_key, place, j0, j1);
  s_rank[which][item] = rank;
  __syncthreads();
  if (tid >= kSmallTile || place >= N) return;
  for (int w = 1; w < kSmallShares; ++w) rank += s_rank[w][item];
  if (!far) keys_out[rank] = s_key[place];
  pos_out[rank] = place;
}

// Where each run of the small sort's equal keys starts, and how many there
// are (runs[0]). IDS: the runs' ids go to `unique`, and how many there are to
// found[0], for the host. Ids that lie far apart have no keys: they are read
// where the sort took them from. Else the runs' rows go to `rows`.
template <bool IDS>
__global__ __launch_bounds__(kSmallThreads) void runs_small_kernel(
    const uint32_t* __restrict__ keys, int N, const int64_t* info,
    const int64_t* __restrict__ ids, const uint32_t* __restrict__ pos,
    uint32_t* starts, uint32_t* runs, uint32_t* rows, int64_t* unique,
    uint32_t* found) {
  __shared__ uint32_t s_count[kSmallWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool far = IDS && info[1] != 0;  // all threads alike
  const int items = (N + kSmallThreads - 1) / kSmallThreads;
  const int i0 = wave * items * 64 + lane;
  uint32_t key[kSmallItems];
  bool first[kSmallItems];
  if (far) {
    int64_t id[kSmallItems], last[kSmallItems];
#pragma unroll
    for (int k = 0; k < kSmallItems; ++k) {
      const int i = i0 + k * 64;
      const bool in = k < items && i < N;
      id[k] = in ? ids[pos[i]] : 0;
      last[k] = in && i > 0 ? ids[pos[i - 1]] : 0;
    }
#pragma unroll
    for (int k = 0; k < kSmallItems; ++k) {
      const int i = i0 + k * 64;
      first[k] = k < items && i < N && (i == 0 || last[k] != id[k]);
    }
  } else {
    uint32_t last[kSmallItems];
#pragma unroll
    for (int k = 0; k < kSmallItems; ++k) {
      const int i = i0 + k * 64;
      const bool in = k < items && i < N;
      key[k] = in ? keys[i] : 0;
      last[k] = in && i > 0 ? keys[i - 1] : 0;
    }
#pragma unroll
    for (int k = 0; k < kSmallItems; ++k) {
      const int i = i0 + k * 64;
      first[k] = k < items && i < N && (i == 0 || last[k] != key[k]);
    }
  }
  uint32_t here = 0, place[kSmallItems];
#pragma unroll
  for (int k = 0; k < kSmallItems; ++k) {
    const uint64_t set = __ballot(first[k]);
    place[k] = here + __builtin_amdgcn_mbcnt_hi(
                          (uint32_t)(set >> 32),
                          __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0));
    here += __popcll(set);
  }
  if (lane == 0) s_count[wave] = here;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int w = 0; w < kSmallWaves; ++w) {
    if (w < wave) before += s_count[w];
    all += s_count[w];
  }
  if (tid == 0) {
    runs[0] = all;
    if constexpr (IDS) found[0] = all;
  }
#pragma unroll
  for (int k = 0; k < kSmallItems; ++k) {
    if (first[k]) {
      const uint32_t at = before + place[k];
      starts[at] = i0 + k * 64;
      if constexpr (IDS)
        unique[at] = far ? ids[pos[i0 + k * 64]]
                         : (int64_t)((uint64_t)info[0] + (uint64_t)key[k]);
      else
        rows[at] = key[k];
    }
  }
}

// Ids over more than 32 bits, up to EDL_SORT_FAR of them. Six passes of the
// radix sort wait for their 18 launches. So chunks of 2048 are sorted as above,
// all at once, and an id's place is the one in its chunk and, for each of the
// other chunks, how many of its ids come before, found by bisection. That grows
// with the square of their number (whole calls by chunks and by passes: 8193
// ids 70 us and 128, 50 thousand 79 and 137, 160 thousand 134 and 154, 200
// thousand 162 and 160).
constexpr int kChunk = 2048, kChunkTile = 128, kChunkGroup = 8;
constexpr int kChunkShares = kSmallThreads / kChunkTile;

__global__ __launch_bounds__(kSmallThreads) void chunk_rank_kernel(
    Keys64 src, int N, uint64_t* __restrict__ keys, uint32_t* __restrict__ pos,
    uint32_t* __restrict__ place) {
  __shared__ __align__(16) uint64_t s_key[kChunk];
  __shared__ uint32_t s_rank[kChunkShares][kChunkTile];
  const int tid = threadIdx.x;
  constexpr int kTiles = kChunk / kChunkTile;
  const int chunk0 = (int)blockIdx.x / kTiles * kChunk;
#pragma unroll
  for (int i = tid; i < kChunk; i += kSmallThreads)
    s_key[i] = chunk0 + i < N ? src(chunk0 + i) : ~0ull;
  __syncthreads();
  const int item = tid % kChunkTile, which = tid / kChunkTile;
  const int at = (int)blockIdx.x % kTiles * kChunkTile + item;
  constexpr int kShare = kChunk / kChunkShares;
  uint32_t rank = rank_among<uint64_t, kChunkTile>(
      s_key, at, which * kShare, (which + 1) * kShare);
  s_rank[which][item] = rank;
  __syncthreads();
  if (tid >= kChunkTile || chunk0 + at >= N) return;
#pragma unroll
  for (int w = 1; w < kChunkShares; ++w) rank += s_rank[w][item];
  keys[chunk0 + rank] = s_key[at];
  pos[chunk0 + rank] = chunk0 + at;
  place[chunk0 + rank] = rank;
}

// places among kChunkGroup chunks, added to those so far: whole numbers, whose
// sum does not depend on the order
__global__ __launch_bounds__(kSmallThreads) void chunk_merge_kernel(
    const uint64_t* __restrict__ keys, int N, uint32_t* place) {
  __shared__ uint64_t s_key[kChunk];
  const int i = (int)blockIdx.x * kSmallThreads + threadIdx.x;
  const int own = (int)blockIdx.x * kSmallThreads / kChunk;
  const int chunks = (N + kChunk - 1) / kChunk;
  const int c0 = (int)blockIdx.y * kChunkGroup;
  const uint64_t key = i < N ? keys[i] : 0;
  uint32_t before = 0;
  for (int c = c0; c < c0 + kChunkGroup && c < chunks; ++c) {
    if (c == own) continue;  // the workgroup alike
    __syncthreads();
#pragma unroll
    for (int k = threadIdx.x; k < kChunk; k += kSmallThreads)
      s_key[k] = c * kChunk + k < N ? keys[c * kChunk + k] : ~0ull;
    __syncthreads();
    const bool first = c < own;  // equal ones of chunks before come before
    int at = 0;
#pragma unroll
    for (int step = kChunk / 2; step > 0; step /= 2) {
      const uint64_t o = s_key[at + step - 1];
      if (o < key || (first && o == key)) at += step;
    }
    const uint64_t o = s_key[at];
    before += at + (o < key || (first && o == key));
  }
  if (i < N && before) atomicAdd(place + i, before);
}

__global__ __launch_bounds__(256) void chunk_move_kernel(
    const uint64_t* __restrict__ keys, const uint32_t* __restrict__ pos,
    const uint32_t* __restrict__ place, int N, uint64_t* __restrict__ keys_out,
    uint32_t* __restrict__ pos_out) {
  const int i = (int)blockIdx.x * 256 + threadIdx.x;
  if (i >= N) return;
  const uint32_t to = place[i];
  keys_out[to] = keys[i];
  pos_out[to] = pos[i];
}

// each workgroup's smallest and largest of ids, for the host: no atomics,
// which thousands of waves would queue up for (100 us for 2.6 million ids,
// against 9)
__global__ __launch_bounds__(256) void range_kernel(
    const int64_t* __restrict__ ids, int64_t N, int64_t* range) {
  __shared__ long long s[2][4];
  long long mn = INT64_MAX, mx = INT64_MIN;
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < N;
       i += 4 * step) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long v = ids[i + u * step < N ? i + u * step : i];
      mn = v < mn ? v : mn;
      mx = v > mx ? v : mx;
    }
  }
  for (int o = 1; o < 64; o <<= 1) {
    const long long a = __shfl_xor(mn, o), b = __shfl_xor(mx, o);
    mn = a < mn ? a : mn;
    mx = b > mx ? b : mx;
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    s[0][wave] = mn;
    s[1][wave] = mx;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) {
      mn = s[0][w] < mn ? s[0][w] : mn;
      mx = s[1][w] > mx ? s[1][w] : mx;
    }
    range[2 * blockIdx.x] = mn;
    range[2 * blockIdx.x + 1] = mx;
  }
}

// ------------------------------ unique ids --------------------------------
// Each item's place among the unique keys: counts of first occurrences by
// tile, their sums, then the places.
template <typename K>
__device__ inline bool first_of(const K* keys, int64_t i) {
  return i == 0 || keys[i] != keys[i - 1];
}

constexpr int kItems = EDL_SORT_TILE / 256, kTile = EDL_SORT_TILE;

template <typename K>
__global__ __launch_bounds__(256) void unique_count_kernel(
    const K* __restrict__ keys, int64_t N, uint32_t* counts) {
  __shared__ uint32_t s4[4];
  uint32_t n = 0;
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = (int64_t)blockIdx.x * kTile + k * 256 + threadIdx.x;
    if (i < N) n += first_of(keys, i);
  }
  uint32_t all;
  block_scan(n, s4, &all);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

template <typename K>
__global__ __launch_bounds__(256) void unique_place_kernel(
    const K* __restrict__ keys, int64_t N, const uint32_t* __restrict__ counts,
    int64_t base, bool turned, uint32_t* __restrict__ place,
    int64_t* __restrict__ unique) {
  __shared__ uint32_t s4[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 =
      (int64_t)blockIdx.x * kTile + wave * (kTile / 4) + lane;
  K key[kItems];
  uint32_t at[kItems], here = 0;
  bool first[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = i0 + k * 64;
    key[k] = i < N ? keys[i] : 0;
    first[k] = i < N && (i == 0 || keys[i - 1] != key[k]);
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const uint64_t set = __ballot(first[k]);
    at[k] = here + __builtin_amdgcn_mbcnt_hi(
                       (uint32_t)(set >> 32),
                       __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0));
    here += __popcll(set);
  }
  if (lane == 0) s4[wave] = here;
  __syncthreads();
  uint32_t before = counts[blockIdx.x];
  for (int w = 0; w < wave; ++w) before += s4[w];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = i0 + k * 64;
    if (i >= N) break;
    const uint32_t p = before + at[k] + first[k] - 1;
    place[i] = p;
    if (first[k])
      unique[p] = turned
                      ? (int64_t)((uint64_t)key[k] ^ 0x8000000000000000ull)
                      : (int64_t)((uint64_t)key[k] + (uint64_t)base);
  }
}

// ------------------------------ summed rows -------------------------------
// The sorted tokens are cut into chunks of a.chunk, whatever the runs
// of equal keys are, so that a frequent id costs no more than rare ones. A
// group of lanes adds its chunk's rows in order, 8 in flight; a run that
// begins and ends in the chunk is written at once. One that goes on past an
// end of the chunk leaves its sum in the workspace, and where it begins the
// join collects the sums of those behind: short runs by a group of lanes of
// a workgroup's first wave, long ones (over kShort chunks) by all of it. Bound
// by the gather: 2.6 million rows of 64 bytes 73 us, 3.6 TB/s (89 with keys
// and positions read one by one), and 13 for the join.
constexpr int kShort = 8;

template <typename T, int VEC>
__global__ __launch_bounds__(256) void segment_kernel(edl_segments a,
                                                      int64_t block0) {
  typedef Vec<T, VEC> V;
  constexpr int U = 8;
  const int lanes = lanes_of(a.D, VEC), pieces = pieces_of(a.D, VEC);
  const int64_t unit = ((block0 + blockIdx.x) * 256 + threadIdx.x) / lanes;
  const int64_t c = unit / pieces;
  const int col =
      ((int)(unit % pieces) * lanes + (threadIdx.x & (lanes - 1))) * VEC;
  const int64_t t0 = c * a.chunk;
  if (t0 >= a.N) return;
  const int64_t t1 = t0 + a.chunk < a.N ? t0 + a.chunk : a.N;
  const bool mine = col < a.D;
  const T* src = static_cast<const T*>(a.src) + (mine ? col : 0);

  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  uint32_t cur = a.keys[t0];
  if (cur >= a.limit) {  // padding, which is sorted behind the rest
    if (col == 0) a.head[c] = a.tail[c] = kNone;
    return;
  }
  bool open = t0 > 0 && a.keys[t0 - 1] == cur;  // begun in a chunk before
  uint32_t head = kNone, tail = kNone;

  auto keep = [&](int which) {
    if (!mine) return;
    float* p = a.part + (c * 2 + which) * a.D + col;
#pragma unroll
    for (int k = 0; k < VEC; ++k) p[k] = acc[k];
  };
  auto write = [&]() {
    if (!mine) return;
    V o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.set(k, acc[k]);
    *reinterpret_cast<decltype(o.v)*>(static_cast<T*>(a.out) +
                                      (int64_t)cur * a.D + col) = o.v;
  };

  for (int64_t t = t0; t < t1; t += U) {
    uint32_t key[U], pos[U], row[U];
    float w[U];
    V v[U];
    // eight at once: t is a multiple of 8, and the arrays' pieces end on
    // borders of 256 bytes
#pragma unroll
    for (int u = 0; u < U; u += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(a.keys + t + u);
      const u32x4 p = *reinterpret_cast<const u32x4*>(a.pos + t + u);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        key[u + q] = k[q];
        pos[u + q] = p[q];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t p = t + u < t1 ? pos[u] : pos[0];
      row[u] = a.L > 1 ? p / (uint32_t)a.L : p;
      w[u] = a.weights ? load_any(a.weights, p, a.w_type) : 1.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].v = *reinterpret_cast<const decltype(v[u].v)*>(
          src + (int64_t)row[u] * a.D);
      w[u] *= a.coef ? a.coef[row[u]] : a.scale;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= t1) break;
      if (key[u] != cur) {
        if (cur < a.limit) {
          if (open) {
            keep(0);
            head = cur;
          } else {
            write();
          }
        }
        cur = key[u];
        open = false;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += w[u] * v[u].get(k);
    }
  }
  const bool goes_on = t1 < a.N && a.keys[t1] == cur;
  if (cur < a.limit) {
    if (open) {
      keep(0);
      head = cur;
    } else if (goes_on) {
      keep(1);
      tail = cur;
    } else {
      write();
    }
  }
  if (col == 0) {
    a.head[c] = head;
    a.tail[c] = tail;
  }
}

// where the small sort has been, and the runs are known: a wave to a run, its
// groups of lanes taking every so-many-th token; one launch in place of three
template <typename T, int VEC>
__global__ __launch_bounds__(256) void segment_run_kernel(edl_segments a,
                                                          int64_t block0) {
  typedef Vec<T, VEC> V;
  constexpr int U = 4;
  const int lanes = lanes_of(a.D, VEC), pieces = pieces_of(a.D, VEC);
  const int lane = threadIdx.x & 63;
  const int64_t unit = ((block0 + blockIdx.x) * 256 + threadIdx.x) >> 6;
  const uint32_t run = (uint32_t)(unit / pieces), runs = *a.runs;
  if (run >= runs) return;
  const int64_t to = a.rows ? a.rows[run] : run;
  if (to >= a.limit) return;
  const int col =
      ((int)(unit % pieces) * lanes + (lane & (lanes - 1))) * VEC;
  const bool mine = col < a.D;
  const T* src = static_cast<const T*>(a.src) + (mine ? col : 0);
  const int groups = 64 / lanes;
  const uint32_t end = run + 1 < runs ? a.starts[run + 1] : (uint32_t)a.N;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  for (uint32_t t = a.starts[run] + lane / lanes; t < end; t += groups * U) {
    uint32_t row[U];
    float w[U];
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = t + u * groups < end;
      const uint32_t p = a.pos[in ? t + u * groups : t];
      row[u] = a.L > 1 ? p / (uint32_t)a.L : p;
      w[u] = a.weights ? load_any(a.weights, p, a.w_type) : 1.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].v = *reinterpret_cast<const decltype(v[u].v)*>(
          src + (int64_t)row[u] * a.D);
      w[u] *= a.coef ? a.coef[row[u]] : a.scale;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u * groups < end) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += w[u] * v[u].get(k);
      }
  }
  for (int o = lanes; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor(acc[k], o);
  if (lane >= lanes || !mine) return;
  V o;
#pragma unroll
  for (int k = 0; k < VEC; ++k) o.set(k, acc[k]);
  *reinterpret_cast<decltype(o.v)*>(static_cast<T*>(a.out) + to * a.D + col) =
      o.v;
}

// how many of the chunks from `in` on begin with this key: they lie together.
// The workgroup looks at 256 places at a time, 80 thousand chunks in 3 rounds
__device__ inline int64_t end_of(const uint32_t* head, uint32_t key,
                                 int64_t in, int64_t out) {
  while (in < out) {
    const int64_t step = (out - in + 255) / 256;
    const int64_t at = in + threadIdx.x * step;
    const int k = __syncthreads_count(at < out && head[at] == key);
    if (k == 0) return in;
    out = in + k * step < out ? in + k * step : out;
    in += (k - 1) * step + 1;
  }
  return in;
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void segment_join_kernel(edl_segments a,
                                                           int64_t chunks,
                                                           int64_t block0) {
  typedef Vec<T, VEC> V;
  constexpr int U = 4;
  __shared__ float s[256 * VEC];
  __shared__ int64_t s_long[64 / kShort + 1];
  __shared__ uint32_t s_longs;
  const int tid = threadIdx.x;
  const int lanes = lanes_of(a.D, VEC), pieces = pieces_of(a.D, VEC);
  const int l_lane = tid & (lanes - 1);
  const int64_t unit = ((block0 + blockIdx.x) * 64 + tid) / lanes;
  if (tid == 0) s_longs = 0;
  __syncthreads();
  const int64_t c0 = unit / pieces;
  const uint32_t key0 = tid < 64 && c0 < chunks ? a.tail[c0] : kNone;
  if (key0 != kNone) {
    const int col = ((int)(unit % pieces) * lanes + l_lane) * VEC;
    int n = 0;  // chunks behind that the run goes on into, up to kShort + 1
    if (c0 + 1 < chunks && a.head[c0 + 1] == key0) {
      bool on = true;
      n = 1;
#pragma unroll
      for (int q = 1; q <= kShort; ++q) {
        const bool in = c0 + 1 + q < chunks;
        on &= a.head[in ? c0 + 1 + q : c0] == key0 && in;
        n += on;
      }
    }
    if (n > kShort) {
      if (l_lane == 0) s_long[atomicAdd(&s_longs, 1u)] = unit;
    } else if (col < a.D) {
      const float* p = a.part + (c0 * 2 + 1) * a.D + col;
      float acc[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = p[k];
      for (int q = 0; q < n; ++q) {
        const float* h = a.part + (c0 + 1 + q) * 2 * a.D + col;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += h[k];
      }
      V o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.set(k, acc[k]);
      *reinterpret_cast<decltype(o.v)*>(static_cast<T*>(a.out) +
                                        (int64_t)key0 * a.D + col) = o.v;
    }
  }
  __syncthreads();
  const int groups = 256 / lanes, g = tid / lanes;
  for (uint32_t at = 0; at < s_longs; ++at) {  // the workgroup together
    const int64_t c = s_long[at] / pieces;
    const int col = ((int)(s_long[at] % pieces) * lanes + l_lane) * VEC;
    const uint32_t key = a.tail[c];
    const int64_t end = end_of(a.head, key, c + 1, chunks);
    float acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    if (col < a.D) {
      for (int64_t q = c + 1 + g; q < end; q += (int64_t)groups * U) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t r = q + (int64_t)u * groups;
          const float* h = a.part + (r < end ? r : q) * 2 * a.D + col;
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[u][k] = r < end ? h[k] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[tid * VEC + k] = acc[k];
    __syncthreads();
    for (int h = groups / 2; h > 0; h >>= 1) {
      if (g < h) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          s[tid * VEC + k] += s[(tid + h * lanes) * VEC + k];
      }
      __syncthreads();
    }
    if (g == 0 && col < a.D) {
      const float* p = a.part + (c * 2 + 1) * a.D + col;
      V o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.set(k, s[tid * VEC + k] + p[k]);
      *reinterpret_cast<decltype(o.v)*>(static_cast<T*>(a.out) +
                                        (int64_t)key * a.D + col) = o.v;
    }
    __syncthreads();
  }
}

// -------------------------------- launches --------------------------------
// a launch holds fewer than 2^32 threads: more go in several
template <typename F>
void in_blocks(int64_t threads, F launch) {
  constexpr int64_t kMost = 1 << 23;
  const int64_t blocks = (threads + 255) / 256;
  for (int64_t b0 = 0; b0 < blocks; b0 += kMost)
    launch((unsigned)(blocks - b0 < kMost ? blocks - b0 : kMost), b0);
}

template <typename T, int VEC>
void launch_lookup(const edl_bag& a, hipStream_t st) {
  const int64_t pieces = pieces_of(a.D, VEC), lanes = lanes_of(a.D, VEC);
  // groups to a bag: until there are 32 waves for each of the 256 CUs, or
  // one eight of ids is left to each
  int subs = 1;
  while (subs * lanes < 64 && subs * 8 < a.L &&
         a.B * pieces * lanes * subs < 256 * 32 * 64)
    subs *= 2;
  in_blocks(a.B * pieces * lanes * subs, [&](unsigned n, int64_t b0) {
    lookup_kernel<T, VEC><<<n, 256, 0, st>>>(a, subs, b0);
  });
}
template <typename T, int VEC>
void launch_weight_grad(const edl_bag& a, hipStream_t st) {
  const int64_t units = a.B * ((a.L + 7) / 8);
  in_blocks(units * lanes_of(a.D, VEC), [&](unsigned n, int64_t b0) {
    weight_grad_kernel<T, VEC><<<n, 256, 0, st>>>(a, b0);
  });
}
template <typename T, int VEC>
void launch_segments(const edl_segments& a, hipStream_t st) {
  if (a.starts) {
    in_blocks(a.N * pieces_of(a.D, VEC) * 64, [&](unsigned n, int64_t b0) {
      segment_run_kernel<T, VEC><<<n, 256, 0, st>>>(a, b0);
    });
    return;
  }
  const int64_t chunks = (a.N + a.chunk - 1) / a.chunk;
  const int64_t threads =
      chunks * pieces_of(a.D, VEC) * lanes_of(a.D, VEC);
  in_blocks(threads, [&](unsigned n, int64_t b0) {
    segment_kernel<T, VEC><<<n, 256, 0, st>>>(a, b0);
  });
  if (chunks == 1) return;
  in_blocks(threads * 4, [&](unsigned n, int64_t b0) {
    segment_join_kernel<T, VEC><<<n, 256, 0, st>>>(a, chunks, b0);
  });
}

#define EDL_BY_TYPE(FN, A, ST)                       \
  if ((A).type == EDL_T_F32) {                       \
    if ((A).vec == 4) FN<float, 4>(A, ST);           \
    else if ((A).vec == 2) FN<float, 2>(A, ST);      \
    else FN<float, 1>(A, ST);                        \
  } else if ((A).type == EDL_T_BF16) {               \
    if ((A).vec == 8) FN<__bf16, 8>(A, ST);          \
    else if ((A).vec == 4) FN<__bf16, 4>(A, ST);     \
    else if ((A).vec == 2) FN<__bf16, 2>(A, ST);     \
    else FN<__bf16, 1>(A, ST);                       \
  } else {                                           \
    if ((A).vec == 8) FN<_Float16, 8>(A, ST);        \
    else if ((A).vec == 4) FN<_Float16, 4>(A, ST);   \
    else if ((A).vec == 2) FN<_Float16, 2>(A, ST);   \
    else FN<_Float16, 1>(A, ST);                     \
  }

// Up to 256 thousand items, a pass less counts for more than the runs in
// which it writes, and tiles of 1024 fill the chip until there are a million.
// Whole gradients of a table of 2^20 - 1 rows, and sums by ids of 27 bits, us:
//   items      Plan4x11   Plan4x9    Plan16x9
//   200,000    61   86    69   82    73  100
//   400,000    60  100    67   98    75  107
//   800,000    85  134    76  130    81  122
//   1,500,000 128  189   107  180   109  161
// The key's width moves where they cross; the borders are between the two.
int sort_plan(int64_t N) {
  return N < 256 * 1024 ? 0 : N < 1024 * 1024 ? 1 : 2;
}
#define EDL_BY_PLAN(N, CALL)                              \
  (sort_plan(N) == 0   ? CALL(Plan4x11)                   \
   : sort_plan(N) == 1 ? CALL(Plan4x9)                    \
                       : CALL(Plan16x9))

template <typename S, bool FIRST, typename P>
int sort_pass(S src, const uint32_t* pos_in, int64_t N, int shift, int bits,
              uint32_t* counts, uint32_t* totals, typename S::K* keys_out,
              uint32_t* pos_out, hipStream_t st, Zeros zeros = {}) {
  constexpr int kTile = P::ITEMS * 256;
  const int tiles = (int)((N + kTile - 1) / kTile);
  const int bins = 1 << bits, fill = zeros.bytes ? kZeroBlocks : 0;
  Zeros half = zeros;  // a part beside each of the two that wait most
  half.bytes = zeros.bytes / 32 * 16;
  zeros.to += half.bytes;
  zeros.bytes -= half.bytes;
  sort_count_kernel<S, P><<<tiles + fill, 256, 0, st>>>(src, N, shift, bits,
                                                        tiles, counts, half);
  sort_offsets_kernel<<<bins, 256, 0, st>>>(counts, tiles, totals);
  sort_move_kernel<S, FIRST, P><<<tiles + fill, 256, 0, st>>>(
      src, pos_in, N, shift, bits, tiles, counts, totals, keys_out, pos_out,
      zeros);
  return (int)hipGetLastError();
}

// Sorts bits `done` to `bits` of keys[at], pos[at] into whichever buffer the
// last pass ends with: returns which, or -1 - error.
template <typename K, typename P>
int sort_rest(int at, int done, int bits, int64_t N, K* const* keys,
              uint32_t* const* pos, uint32_t* counts, uint32_t* totals,
              hipStream_t st) {
  while (done < bits) {
    const int left = (bits - done + P::BITS - 1) / P::BITS;
    const int b = (bits - done + left - 1) / left;
    const int rc = sort_pass<KeysOf<K>, false, P>(
        KeysOf<K>{keys[at]}, pos[at], N, done, b, counts, totals,
        keys[at ^ 1], pos[at ^ 1], st);
    if (rc) return -1 - rc;
    at ^= 1;
    done += b;
  }
  return at;
}
// all of it; the first pass, into keys[0], makes the keys from src
template <typename S, typename P>
int sort_by(S src, int64_t N, int bits, typename S::K* const* keys,
            uint32_t* const* pos, uint32_t* counts, uint32_t* totals,
            hipStream_t st, Zeros zeros) {
  const int passes = (bits + P::BITS - 1) / P::BITS;
  const int b = (bits + passes - 1) / passes;
  const int rc = sort_pass<S, true, P>(src, nullptr, N, 0, b, counts, totals,
                                       keys[0], pos[0], st, zeros);
  if (rc) return -1 - rc;
  return sort_rest<typename S::K, P>(0, b, bits, N, keys, pos, counts, totals,
                                     st);
}
template <typename S>
int sort_all(S src, int64_t N, int bits, typename S::K* const* keys,
             uint32_t* const* pos, uint32_t* counts, uint32_t* totals,
             hipStream_t st, Zeros zeros = {}) {
#define EDL_SORT_BY(P) \
  sort_by<S, P>(src, N, bits, keys, pos, counts, totals, st, zeros)
  return EDL_BY_PLAN(N, EDL_SORT_BY);
#undef EDL_SORT_BY
}

template <typename K>
int unique_all(const K* keys, int64_t N, uint32_t* counts, uint32_t* found,
               int64_t base, bool turned, uint32_t* place, int64_t* unique,
               hipStream_t st) {
  const int tiles = (int)((N + kTile - 1) / kTile);
  unique_count_kernel<K><<<tiles, 256, 0, st>>>(keys, N, counts);
  sort_offsets_kernel<<<1, 256, 0, st>>>(counts, tiles, found);
  unique_place_kernel<K><<<tiles, 256, 0, st>>>(keys, N, counts, base, turned,
                                                place, unique);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int edl_lookup(const edl_bag* a, hipStream_t st) {
  EDL_BY_TYPE(launch_lookup, *a, st)
  return (int)hipGetLastError();
}

extern "C" int edl_lookup_weight_grad(const edl_bag* a, hipStream_t st) {
  EDL_BY_TYPE(launch_weight_grad, *a, st)
  return (int)hipGetLastError();
}

extern "C" int edl_segment_sums(const edl_segments* a, hipStream_t st) {
  EDL_BY_TYPE(launch_segments, *a, st)
  return (int)hipGetLastError();
}

// Sorts the ids of a table of V rows, those without a row behind the rest,
// and fills `zeros` with them. Returns which of the two buffers holds the
// result, or -1 - error.
extern "C" int edl_sort_rows(const void* ids, int ids64, int64_t V, int64_t N,
                             uint32_t* const* keys, uint32_t* const* pos,
                             uint32_t* counts, uint32_t* totals, void* zeros,
                             int64_t zero_bytes, hipStream_t st) {
  int bits = 1;
  while (bits < 32 && (V >> bits) != 0) ++bits;
  Keys32 src{ids, ids64 != 0, V};
  return sort_all(src, N, bits, keys, pos, counts, totals, st,
                  Zeros{static_cast<uint8_t*>(zeros), zero_bytes});
}

// chunks for the segment kernels: as long as they leave 16 waves for each of
// the 256 CUs, from 8 to 32 tokens
extern "C" int edl_segment_chunk(int64_t N, int D, int vec) {
  const int64_t per = (int64_t)pieces_of(D, vec) * lanes_of(D, vec);
  int chunk = 32;
  while (chunk > 8 && N / chunk * per < 256 * 16 * 64) chunk /= 2;
  return chunk;
}

// how many counts a sort of N items needs
extern "C" int64_t edl_sort_counts(int64_t N) {
#define EDL_COUNTS(P) \
  ((N + P::ITEMS * 256 - 1) / (P::ITEMS * 256) << P::BITS)
  return EDL_BY_PLAN(N, EDL_COUNTS);
#undef EDL_COUNTS
}

// the small sorts, and their runs: see the kernels
extern "C" int edl_sort_rows_small(const void* ids, int ids64, int64_t V,
                                   int64_t N, uint32_t* keys, uint32_t* pos,
                                   uint32_t* starts, uint32_t* runs,
                                   uint32_t* rows, void* zeros,
                                   int64_t zero_bytes, hipStream_t st) {
  const int tiles = (int)((N + kSmallTile - 1) / kSmallTile);
  const int64_t fill = std::min<int64_t>(
      (zero_bytes + kSmallThreads * 16 - 1) / (kSmallThreads * 16),
      kZeroBlocks * 256 / kSmallThreads);
  rank_small_kernel<Keys32, false>
      <<<tiles + (int)fill, kSmallThreads, 0, st>>>(
          Keys32{ids, ids64 != 0, V}, (int)N, keys, pos, nullptr, tiles,
          Zeros{static_cast<uint8_t*>(zeros), zero_bytes});
  runs_small_kernel<false><<<1, kSmallThreads, 0, st>>>(
      keys, (int)N, nullptr, nullptr, nullptr, starts, runs, rows, nullptr,
      nullptr);
  return (int)hipGetLastError();
}
extern "C" int edl_sort_ids_small(const int64_t* ids, int64_t N,
                                  uint32_t* keys, uint32_t* pos, int64_t* info,
                                  uint32_t* starts, uint32_t* runs,
                                  int64_t* unique, uint32_t* found,
                                  hipStream_t st) {
  const int tiles = (int)((N + kSmallTile - 1) / kSmallTile);
  rank_small_kernel<Keys32Of, true><<<tiles, kSmallThreads, 0, st>>>(
      Keys32Of{ids}, (int)N, keys, pos, info, tiles, Zeros{});
  runs_small_kernel<true><<<1, kSmallThreads, 0, st>>>(
      keys, (int)N, info, ids, pos, starts, runs, nullptr, unique, found);
  return (int)hipGetLastError();
}

// pairs of smallest and largest, one for each of EDL_RANGE_PARTS parts
extern "C" int edl_ids_range(const int64_t* ids, int64_t N, int64_t* range,
                             hipStream_t st) {
  range_kernel<<<EDL_RANGE_PARTS, 256, 0, st>>>(ids, N, range);
  return (int)hipGetLastError();
}

// Ids whose bits from the 32nd up are all the same, by their low bits. The
// first pass, over `first` bits into keys[0], needs not know how many: it is
// launched while the host still waits for their range.
extern "C" int edl_sort_ids32_first(const int64_t* ids, int first, int64_t N,
                                    uint32_t* const* keys,
                                    uint32_t* const* pos, uint32_t* counts,
                                    uint32_t* totals, hipStream_t st) {
  Keys32Of src{ids};
#define EDL_FIRST(P)                                                        \
  sort_pass<Keys32Of, true, P>(src, nullptr, N, 0, first, counts, totals,   \
                               keys[0], pos[0], st)
  return EDL_BY_PLAN(N, EDL_FIRST);
#undef EDL_FIRST
}
extern "C" int edl_sort_ids32_rest(int first, int bits, int64_t N,
                                   uint32_t* const* keys, uint32_t* const* pos,
                                   uint32_t* counts, uint32_t* totals,
                                   hipStream_t st) {
#define EDL_REST(P)                                                         \
  sort_rest<uint32_t, P>(0, first, bits, N, keys, pos, counts, totals, st)
  return EDL_BY_PLAN(N, EDL_REST);
#undef EDL_REST
}

extern "C" int edl_sort_ids64(const int64_t* ids, int64_t N,
                              uint64_t* const* keys, uint32_t* const* pos,
                              uint32_t* counts, uint32_t* totals,
                              hipStream_t st) {
  if (N > EDL_SORT_FAR)
    return sort_all(Keys64{ids}, N, 64, keys, pos, counts, totals, st);
  static_assert(EDL_SORT_FAR < 256 * 1024, "counts have room for the places");
  const int n = (int)N, chunks = (n + kChunk - 1) / kChunk;
  uint32_t* place = counts;
  chunk_rank_kernel<<<(n + kChunkTile - 1) / kChunkTile, kSmallThreads, 0,
                      st>>>(Keys64{ids}, n, keys[0], pos[0], place);
  chunk_merge_kernel<<<dim3((n + kSmallThreads - 1) / kSmallThreads,
                            (chunks + kChunkGroup - 1) / kChunkGroup),
                       kSmallThreads, 0, st>>>(keys[0], n, place);
  chunk_move_kernel<<<(n + 255) / 256, 256, 0, st>>>(keys[0], pos[0], place, n,
                                                     keys[1], pos[1]);
  const int rc = (int)hipGetLastError();
  return rc ? -1 - rc : 1;
}

extern "C" int edl_unique32(const uint32_t* keys, int64_t N, uint32_t* counts,
                            uint32_t* found, int64_t base, uint32_t* place,
                            int64_t* unique, hipStream_t st) {
  return unique_all(keys, N, counts, found, base, false, place, unique, st);
}

extern "C" int edl_unique64(const uint64_t* keys, int64_t N, uint32_t* counts,
                            uint32_t* found, uint32_t* place, int64_t* unique,
                            hipStream_t st) {
  return unique_all(keys, N, counts, found, 0, true, place, unique, st);
}
