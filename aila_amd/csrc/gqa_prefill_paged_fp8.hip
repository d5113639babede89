// Causal GQA attention of a ragged batch over the 8-bit paged cache (gfx950).
//
//   o_i = sum_j softmax_j(q_i . K_j / sqrt(D)) V_j over the rows j <= L - n + i
//
// for the n tokens of each request. The query rows of a KV head are (token,
// head) pairs, token-major, in tiles of 128: all query heads that read a KV
// head share its rows, so a code is converted once for all of them.
//
// One workgroup walks a tile with two groups of 4 waves, each group every
// second key tile and each wave 32 query rows; their softmax states meet in LDS
// at the end. Products on v_mfma_f32_32x32x16_bf16:
//   S^T = K Q^T     A = 32 keys (LDS), B = the wave's 32 query rows (registers)
//   O^T += V^T P^T  A = 32 head dims (LDS), B = P, in the registers where S^T
//                   left it: lane (l % 32, h = l / 32) holds keys 8 a + 4 h + c
//                   (a, c < 4) of its column, so step s of a 32-key tile takes
//                   keys 16 s + 4 h + {0..3, 8..11} and V is laid out for that.
//
// Codes come by DMA into LDS, two tiles ahead. A group's vector phase turns
// them into bf16 operands - times the block's scale, which the conversion
// applies for free and exactly - in the order in which the waves read them:
// every operand is one contiguous KiB a wave. V is transposed on the way: a
// thread takes 8 keys x 4 dims and pairs their bytes with v_perm.
//
// The groups alternate: while one is in its matrix phase M(j) (O += V_{j-1}
// P_{j-1}, S_j = K_j Q), the other is in its vector phase V(j) (softmax of S_j,
// conversion of V_j and K_{j+1}), so each SIMD's matrix core and vector ALU are
// both fed, by one wave each. A phase is 1850 cycles at D = 256 (32 keys), where
// the operand reads of the matrix phase bound it, and 2130 at D = 128 (64 keys),
// where the vector phase does, for 1056 cycles of products.
//
// 8191 tokens, 16 / 4 heads, D = 256: 505-530 us (1.04-1.09 PFLOP/s; a large bf16
// product reaches 1.19 here); 2048 tokens, 32 / 8, D = 128: 47-49 us; 250 tokens after
// 7900, D = 256: 50-51 us with 7 us of merge; 3 prompts of up to 600 tokens after 3000
// rows beside 29 single tokens, 40 / 8, D = 128: 138-141 us with 5.5 us of plan and
// 4.7 us of merge.
#include "paged_fp8.hpp"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace aila {
namespace {

constexpr int kGroupWaves = 4;
constexpr int kGroup = 64 * kGroupWaves;   // threads of a group
constexpr int kThreads = 2 * kGroup;
constexpr int kRows = 32 * kGroupWaves;    // query rows of a tile
constexpr int kMaxSequences = 4096;
constexpr int kCus = 256;
constexpr int kNoKey = 0x7fffffff;
// A tile of so few rows is walked by single waves (us a call, so / as the others, in a
// graph that changes its inputs. 32 requests of 1 token after up to 3000 rows: 32 / 8,
// D = 64 28.1 / 50.3, D = 128 42.4 / 65.8, 16 / 4, D = 256 58.5 / 74.0; 8 after up to
// 30000, D = 256 101.6 / 129.2; one after 5000, D = 128 20.2 / 25.4, D = 256 26.8 / 29.2;
// its 4 tokens after 30000, 16 rows, D = 256 47.0 / 45.7, the one case that loses).
constexpr int kThinRows = 16;

struct Fp8PrefillArgs {
  const bf16* q;
  long q_stride;
  bf16* out;
  float* part;           // records of the tiles whose keys are split
  const int* query_start;
  const int* seq_lens;
  int T, B, Hq, group;
  int max_len;
  int lanes;             // workgroups per KV head
  int splits;            // one request: key runs a tile is cut into
  int* plan;             // several requests: the items' list (null: one request)
  float scale_log2;
};

// The list of a ragged batch's items: counts, the items in order of falling
// size, and the tiles whose keys are cut.
constexpr int kPlanHead = 16;
struct PlanItem { int b, r0, t0, t1, rec; };
struct PlanCut { int b, r0, rec, cuts; };
__host__ __device__ inline long plan_items(long T, int B, int group, int lanes) {
  return (T * group + kRows - 1) / kRows + B + lanes;
}
__host__ __device__ inline long plan_bytes(long T, int B, int group, int lanes) {
  const long n = kPlanHead * 4 + plan_items(T, B, group, lanes) * static_cast<long>(sizeof(PlanItem)) +
                 lanes * static_cast<long>(sizeof(PlanCut));
  return (n + 255) / 256 * 256;
}

template <int D>
struct Cfg {
  static constexpr int BN = D == 256 ? 32 : 64;   // keys of a tile
  static constexpr int KT = BN / 32;              // 32-key parts
  static constexpr int NB = BN / kScaleRows;      // blocks
  static constexpr int STEPS = D / 16;            // MFMA steps over D (S^T)
  static constexpr int DT = D / 32;               // 32-dim parts (O^T)
  static constexpr int CH = D / 16;               // 16-byte pieces of a row of codes
  static constexpr int OPS = BN * D * 2;          // bytes of a tile as operands
  static constexpr int RAW = BN * D;              // bytes of a tile as codes
  static constexpr int DMA = RAW / (1024 * kGroupWaves);   // DMA instructions a wave and tile
  static constexpr int KI = BN * CH / kGroup;     // 16-code pieces of K a thread converts
  static constexpr int AHEAD = D == 256 ? 3 : 4;  // LDS operand reads in flight ahead of their MFMAs
  static constexpr int SEG = D == 256 ? 704 : 2048;   // blocks of a segment of keys, looked up at once
  static constexpr int QL = D == 256 ? 5 : 0;     // MFMA steps whose query operand is kept in LDS: the registers do not hold it
  static constexpr int LDS = 2 * (2 * OPS + 4 * RAW);
  static constexpr int XR = D == 256 ? 2 : 1;     // rounds in which the groups exchange their outputs
  static_assert(2 * OPS >= kGroupWaves * DT / XR * 2 * 1024, "half a group's outputs fit its operands' place");
  static constexpr int REC = kRows * (D + 2);     // floats of a record: {o[rows][D], {m, l}[rows]}
};

__device__ __forceinline__ f32x16 mfma32(const bf16x8_t& a, const bf16x8_t& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Max over lanes l and l ^ 32.
__device__ __forceinline__ float half_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// x, as a value the compiler cannot follow: what is made of it inside a loop is
// made there again, a few instructions, and not kept in registers (or spilled)
// over all loops around it.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// acc + the two bf16 of x.
__device__ __forceinline__ float add_pair(uint32_t x, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc, false);
}

__device__ __forceinline__ void pin(u32x4& x) { asm volatile("" : "+v"(x)); }

// Head dim of row m of output part dt (the order in which V's bytes pair up).
template <int D>
__device__ __forceinline__ int out_dim(int dt, int m) {
  if constexpr (D == 64) return 4 * (m & 15) + 2 * dt + (m >> 4);
  else return 4 * m + (dt & 3) + 128 * (dt >> 2);
}
// Part and row of byte j of dim quad dq.
template <int D>
__device__ __forceinline__ void out_slot(int dq, int j, int* dt, int* m) {
  if constexpr (D == 64) {
    *dt = j >> 1;
    *m = dq + 16 * (j & 1);
  } else {
    *dt = j + 4 * (dq >> 5);
    *m = dq & 31;
  }
}

// K codes of a row lie in LDS with their 16-byte pieces exchanged, so that 8
// neighbouring rows' reads of one piece fall into different banks.
template <int D>
__device__ __forceinline__ int piece_swizzle(int r) {
  return D == 64 ? (r >> 1) & 3 : r & 7;
}

// What a workgroup does next: a tile of query rows and a run of its keys.
struct Item {
  int b, r0;          // request, first query row
  int t0, t1;         // key tiles
  int rec;            // record, -1: the run is the tile's only one
  int q0, n, len;     // the request's first token, tokens, rows
};

__device__ __forceinline__ void load_request(const Fp8PrefillArgs& a, int b, Item* it) {
  it->b = b;
  it->q0 = min(max(a.query_start[b], 0), a.T);
  it->n = max(min(max(a.query_start[b + 1], 0), a.T) - it->q0, 0);
  it->len = min(max(a.seq_lens[b], 0), a.max_len);
}

// Keys that some row of the tile attends.
__device__ __forceinline__ int tile_end(const Fp8PrefillArgs& a, const Item& it) {
  return max(it.len - it.n + min(it.n - 1, (it.r0 + kRows - 1) / a.group) + 1, 0);
}

// Item `index` of a KV head; false: there is none. One request: tiles with more
// keys first, their keys in `splits` equal runs.
template <int D>
__device__ __forceinline__ bool get_item(const Fp8PrefillArgs& a, int index, Item* it) {
  if (a.plan != nullptr) {
    if (index >= a.plan[0]) return false;
    const PlanItem x = reinterpret_cast<const PlanItem*>(a.plan + kPlanHead)[index];
    load_request(a, x.b, it);
    it->r0 = x.r0;
    it->t0 = x.t0;
    it->t1 = x.t1;
    it->rec = x.rec;
    return true;
  }
  load_request(a, 0, it);
  const int tiles = (it->n * a.group + kRows - 1) / kRows;
  const int rank = a.splits > 1 ? index / a.splits : index, cut = index - rank * a.splits;
  if (rank >= tiles) return false;
  it->r0 = (tiles - 1 - rank) * kRows;
  const unsigned kt = (tile_end(a, *it) + Cfg<D>::BN - 1) / Cfg<D>::BN;
  it->t0 = 0;
  it->t1 = kt;
  it->rec = -1;
  if (a.splits > 1) {
    const unsigned n = a.splits, each = kt / n, rest = kt % n;   // run i begins at floor(i kt / n)
    it->t0 = each * cut + rest * cut / n;
    it->t1 = each * (cut + 1) + rest * (cut + 1) / n;
    it->rec = index;
  }
  return true;
}

// The items of a ragged batch. Each workgroup of a KV head should get the same
// number of key tiles: a tile of query rows with more of them than that share
// is cut into equal runs of at most a share, and the items are sorted by size,
// so that the workgroups, which take them forth and back, fill up evenly.
// Shorter runs cost more in records than they gain: key tiles in a batch, keys of one
// request (us, D = 128, 32 / 8: 8 requests of 32 tokens and up to 1200 rows, 4 tiles
// 35.3, 8 31.4; one of 32 after 1200, 256 keys 16.6, 512 19.4; of 5000, 22.3 and 22.5).
constexpr int kMinRun = 8, kMinKeys = 256;

template <int NT, typename T>
__device__ __forceinline__ T plan_scan(T x, T* s_wave, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) before += s_wave[w];
    all += s_wave[w];
  }
  *total = all;
  return x + before;   // inclusive
}

template <int NT>
__global__ __launch_bounds__(NT) void gqa_prefill_paged_fp8_plan_kernel(Fp8PrefillArgs a, int key_tile) {
  constexpr int kBuckets = NT;
  extern __shared__ int s_dyn_plan[];
  int* s_first = s_dyn_plan;          // [B + 1] first tile of each request
  int* s_n = s_first + a.B + 1;       // [B] tokens
  int* s_len = s_n + a.B;             // [B] rows
  __shared__ int s_wave[NT / 64];
  __shared__ long s_wave_l[NT / 64];
  __shared__ int s_bucket[kBuckets];
  __shared__ int s_share[16], s_runs[16], s_cost[kCus];
  const int tid = threadIdx.x;
  PlanItem* items = reinterpret_cast<PlanItem*>(a.plan + kPlanHead);
  PlanCut* cuts_of = reinterpret_cast<PlanCut*>(items + plan_items(a.T, a.B, a.group, a.lanes));
  s_bucket[tid] = 0;
  if (tid == 0) s_first[0] = 0;
  // malformed starts may overlap: no more tiles than the list holds
  const long most = plan_items(a.T, a.B, a.group, 0);
  long all_tiles = 0;
  for (int b0 = 0; b0 < a.B; b0 += NT) {
    const int b = b0 + tid;
    Item it{};
    if (b < a.B) load_request(a, b, &it);
    long all;
    const long incl = all_tiles + plan_scan<NT, long>((it.n * a.group + kRows - 1) / kRows, s_wave_l, &all);
    if (b < a.B) {
      s_first[b + 1] = static_cast<int>(min(incl, most));
      s_n[b] = it.n;
      s_len[b] = it.len;
    }
    all_tiles += all;
  }
  const int tiles = static_cast<int>(min(all_tiles, most));
  __syncthreads();
  // Tile f: its request, first row, key tiles and what walking them costs, in
  // quarters of a key tile: one of at most kThinRows rows is walked by single
  // waves, each its own keys.
  struct Tile { int b, r0, kt, cost; };
  auto tile = [&](int f) __attribute__((always_inline)) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_first[mid] <= f) lo = mid; else hi = mid;
    }
    Tile x;
    x.b = lo;
    x.r0 = (f - s_first[lo]) * kRows;
    Item it{};
    it.n = s_n[lo];
    it.len = s_len[lo];
    it.r0 = x.r0;
    x.kt = (tile_end(a, it) + key_tile - 1) / key_tile;
    x.cost = it.n * a.group - x.r0 <= kThinRows ? x.kt : 4 * x.kt;
    return x;
  };
  Tile mine{};      // the first round's, which is all there are as a rule
  if (tid < tiles) mine = tile(tid);
  auto tile_at = [&](int f) __attribute__((always_inline)) { return f < NT ? mine : tile(f); };
  long sum = 0;
  for (int f0 = 0; f0 < tiles; f0 += NT) {
    const int f = f0 + tid;
    long all;
    plan_scan<NT, long>(f < tiles ? tile_at(f).cost : 0, s_wave_l, &all);
    sum += all;
  }
  // The share: an equal part of the whole, but where all tiles can run at once, the
  // smallest of some that leaves no more runs than workgroups (a run too many would
  // wait for another to end: 8 requests of 32 tokens and up to 5000 rows, 16 / 4, D =
  // 256: 85 -> 57 us). The last always does: a run a tile, and sum / share more.
  // (No tile costs 2^28: T * group and max_len are at most 2^30.)
  constexpr int kShares = 9;
  if (tid < kShares) {
    const long even = max(4L * kMinRun, (sum + a.lanes - 1) / a.lanes);
    const long x = tid < kShares - 1 ? even + even * tid / 8 : max(even, sum / max(1, a.lanes - tiles) + 1);
    s_share[tid] = static_cast<int>(min(x, 1L << 28));
  }
  const bool one_round = tiles <= a.lanes;      // fewer than the threads
  if (one_round && tid < tiles) s_cost[tid] = mine.cost;
  __syncthreads();
  int share = s_share[0];
  if (one_round) {
    for (int k = tid >> 6; k < kShares; k += NT / 64) {
      int runs = 0;
      for (int f = tid & 63; f < tiles; f += 64) runs += max(1, (s_cost[f] + s_share[k] - 1) / s_share[k]);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) runs += __shfl_xor(runs, off);
      if ((tid & 63) == 0) s_runs[k] = runs;
    }
    __syncthreads();
    int pick = INT_MAX;
#pragma unroll
    for (int k = 0; k < kShares; ++k)
      if (s_runs[k] <= a.lanes) pick = min(pick, s_share[k]);
    if (pick != INT_MAX) share = pick;
  }
  auto cuts_for = [&](const Tile& x) __attribute__((always_inline)) { return max(1, (x.cost + share - 1) / share); };
  // run i of a tile's key tiles, large runs' buckets first
  auto run_begin = [&](const Tile& x, int cuts, int i) __attribute__((always_inline)) {
    return x.kt / cuts * i + x.kt % cuts * i / cuts;
  };
  auto bucket = [&](const Tile& x, int cuts) __attribute__((always_inline)) {
    return kBuckets - 1 - static_cast<int>(static_cast<long>(x.cost / cuts) * (kBuckets - 1) / share);
  };
  for (int f = tid; f < tiles; f += NT) {
    const Tile x = tile_at(f);
    const int cuts = cuts_for(x);
    atomicAdd(&s_bucket[bucket(x, cuts)], cuts);
  }
  __syncthreads();
  const int count = s_bucket[tid];
  int total;
  const int incl = plan_scan<NT, int>(count, s_wave, &total);
  s_bucket[tid] = incl - count;
  __syncthreads();
  // Which workgroup an item goes to depends on the order within a bucket, its
  // result does not: records are numbered by the tiles' order.
  int recs = 0, cut_tiles = 0;
  for (int f0 = 0; f0 < tiles; f0 += NT) {
    const int f = f0 + tid;
    Tile x{};
    int cuts = 0;
    if (f < tiles) {
      x = tile_at(f);
      cuts = cuts_for(x);
    }
    // both sums in one: fewer than 2^15 tiles are cut, into fewer than 2^16 runs
    const int cut = cuts > 1 ? cuts << 15 | 1 : 0;
    int all;
    const int before = plan_scan<NT, int>(cut, s_wave, &all) - cut;
    const int rec = recs + (before >> 15), slot = cut_tiles + (before & 0x7fff);
    recs += all >> 15;
    cut_tiles += all & 0x7fff;
    if (cut) cuts_of[slot] = PlanCut{x.b, x.r0, rec, cuts};
    if (cuts > 0) {
      int at = atomicAdd(&s_bucket[bucket(x, cuts)], cuts);
      for (int i = 0; i < cuts; ++i, ++at)
        items[at] = PlanItem{x.b, x.r0, run_begin(x, cuts, i), run_begin(x, cuts, i + 1), cut ? rec + i : -1};
    }
  }
  if (tid == 0) {
    a.plan[0] = total;
    a.plan[1] = cut_tiles;
  }
}

// Place in a record of head dim d of query row r < 32.
template <int D>
__device__ __forceinline__ int record_at(int r, int d) {
  const int j = d & 3;
  const int dt = D == 64 ? j >> 1 : j + 4 * (d >> 7), m = D == 64 ? (d >> 2) + 16 * (j & 1) : (d & 127) >> 2;
  return ((dt * 4 + (m >> 3)) * 64 + (m >> 2 & 1) * 32 + r) * 4 + (m & 3);
}

// A tile of up to 16 rows (a decoding request's token, the rest of a prompt): no
// use of the codes but one, so nothing is staged. Each of the workgroup's 8
// waves walks every eighth strip of 32 keys as the decode kernel does, and
// their states meet in LDS (s_o: 16 * 8 * D floats).
template <int D>
__device__ __forceinline__ void thin_item(const PagedFp8& c, const Fp8PrefillArgs& a, const Item& it, int kvh, float* s_o,
                                          float* s_ml) {
  constexpr int kWaves = kThreads / 64;
  constexpr int kDepth = D == 256 ? 1 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, g4 = lane >> 4;
  const int rows = it.n * a.group - it.r0;
  const int row = it.r0 + min(m16, rows - 1);
  const int tok = row / a.group;
  const int lim = max(it.len - it.n + tok + 1, 0);
  const int first = max(it.len - it.n + it.r0 / a.group + 1, 0);   // keys that every row attends
  const bf16* src = a.q + static_cast<size_t>(it.q0 + tok) * a.q_stride + static_cast<size_t>(kvh * a.group + row - tok * a.group) * D;
  bf16x8_t q[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) q[ks] = as_bf16x8(ld16(src + 64 * (ks >> 1) + 16 * g4 + 8 * (ks & 1)));
  Column<D> col;
  clear_column(col);
  const int row0 = it.t0 * Cfg<D>::BN + 32 * wave;
  const int end = min(it.t1 * Cfg<D>::BN, tile_end(a, it));
  const int ns = row0 < end ? (end - row0 + 32 * kWaves - 1) / (32 * kWaves) : 0;
  const int blk_end = (end + kScaleRows - 1) / kScaleRows;
  for (int n0 = 0; n0 < ns; n0 += 32) {
    const BlockRef mine = block_ref(c, it.b, kvh, row0 / kScaleRows + (n0 + (lane >> 1)) * (2 * kWaves) + (lane & 1), blk_end);
    const int n1 = min(ns - n0, 32);
    auto load = [&](Strip<D>& s, int n) __attribute__((always_inline)) {
      const bool in = n < n1;
      const int ba = __builtin_amdgcn_readlane(mine.bid, 2 * n & 63), bb = __builtin_amdgcn_readlane(mine.bid, (2 * n + 1) & 63);
      load_strip<D, true>(s, c, in ? ba : -1, in ? bb : -1, m16, g4);
    };
    Strip<D> s[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) load(s[i], i);
    for (int n = 0; n < n1; n += kDepth) {
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        if (n + i < n1) {
          load(s[(i + kDepth - 1) % kDepth], n + i + kDepth - 1);
          const int ba = __builtin_amdgcn_readlane(mine.bid, 2 * (n + i)), bb = __builtin_amdgcn_readlane(mine.bid, 2 * (n + i) + 1);
          const int at = row0 + (n0 + n + i) * 32 * kWaves;
          strip_step<D>(col, s[i], q, readlane_f(mine.ks, 2 * (n + i)) * a.scale_log2, readlane_f(mine.ks, 2 * (n + i) + 1) * a.scale_log2,
                        readlane_f(mine.vs, 2 * (n + i)), readlane_f(mine.vs, 2 * (n + i) + 1),
                        at + 32 > min(end, first) || (ba | bb) < 0, at, min(lim, end), ba >= 0, bb >= 0, g4);
        }
      }
    }
  }
  const float l = xrow4_sum(col.l);
  __syncthreads();     // the item before has been written
  float* mine_o = s_o + (wave * 16 + m16) * D;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int t = 0; t < D / 16; ++t) mine_o[(D / 16) * (4 * g4 + i) + t] = col.acc[t][i];
  }
  if (g4 == 0) {
    s_ml[(wave * 16 + m16) * 2] = col.m;
    s_ml[(wave * 16 + m16) * 2 + 1] = l;
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < rows * D; idx += kThreads) {
    const int r = idx / D, d = idx % D;
    float M = -INFINITY, A = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_ml[(w * 16 + r) * 2]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = s_ml[(w * 16 + r) * 2];
      const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
      A += f * s_o[(w * 16 + r) * D + d];
      L += f * s_ml[(w * 16 + r) * 2 + 1];
    }
    if (it.rec >= 0) {
      float* rec = a.part + (static_cast<size_t>(it.rec) * c.Hkv + kvh) * Cfg<D>::REC;
      rec[record_at<D>(r, d)] = A;
      if (d == 0) {
        rec[kRows * D + r * 2] = M;
        rec[kRows * D + r * 2 + 1] = L;
      }
    } else {
      const int rr = it.r0 + r, tk = rr / a.group;
      a.out[(static_cast<size_t>(it.q0 + tk) * a.Hq + kvh * a.group + rr - tk * a.group) * D + d] = f2bf(L == 0.f ? 0.f : A / L);
    }
  }
  __syncthreads();     // LDS is the next item's
}

// THIN: the items may be thin ones. (A kernel that never meets one is a variant of
// its own: the thin walk's registers cost the other's loop 5-9%.)
template <int D, bool THIN>
__global__ __launch_bounds__(kThreads, 1) void gqa_prefill_paged_fp8_kernel(PagedFp8 c, Fp8PrefillArgs a) {
  using C = Cfg<D>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char s_dyn[];
  __shared__ int s_nan[D];      // first masked-tile key whose V holds NaN in this dim
  __shared__ int s_any_nan;
  __shared__ float s_ml[2][kRows][2];
  // Blocks of the segment of keys being walked: index in the pool (-1: none), scales.
  __shared__ __attribute__((aligned(16))) int s_bid[C::SEG];
  __shared__ float s_ks[C::SEG], s_vs[C::SEG];
  __shared__ __attribute__((aligned(16))) unsigned char s_q[(C::QL ? kGroupWaves * C::QL : 1) * 1024];
  const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / kGroup);
  const int t = threadIdx.x % kGroup, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  // operands of both groups (the exchange of their outputs at the end), then codes
  unsigned char* k_ops = s_dyn + grp * 2 * C::OPS;
  unsigned char* v_ops = k_ops + C::OPS;
  unsigned char* k_raw = s_dyn + 4 * C::OPS + grp * 4 * C::RAW;   // two tiles
  unsigned char* v_raw = k_raw + 2 * C::RAW;                      // two tiles
  // This thread's places, in bytes: of its codes in a page (K: pieces exchanged;
  // V: lane * 16), of the codes it converts, and of the operands it makes.
  constexpr int kKib = kScaleRows * D / 1024;          // KiB of a block
  const unsigned uh = threadIdx.x % kGroup, ul = threadIdx.x & 63;
  const unsigned kr = (64 / C::CH) * (wave % kKib) + ul / C::CH;     // row in its block
  const int k_off = (ul / C::CH) * D + ((ul % C::CH) ^ piece_swizzle<D>(kr)) * 16;
  const unsigned cr = uh % C::BN, cs = uh / C::BN;     // K: row of the tile, first piece
  const int k_from = cr * D + ((cs ^ piece_swizzle<D>(cr)) << 4);
  const int k_to = ((cr / 32 * C::STEPS + cs) * 64 + cr % 32) * 16;
  const unsigned oc = uh / (D / 4), dq = uh % (D / 4);  // V: octet of keys, quad of dims
  const int v_from = (16 * (oc >> 1) + 4 * (oc & 1)) * D + 4 * dq;
  int v_dt, v_row;
  out_slot<D>(dq, 0, &v_dt, &v_row);
  const int v_to = (((oc >> 1) * C::DT + v_dt) * 64 + (oc & 1) * 32 + v_row) * 16;
  const int kvh = static_cast<int>(blockIdx.x) % c.Hkv, wl = static_cast<int>(blockIdx.x) / c.Hkv;

  // group 1 walks the odd tiles of the segment; block 0 of tile j
  auto first_block = [&](int j) __attribute__((always_inline)) { return (2 * j + grp) * C::NB; };

  // ---- DMA of a tile's codes -----------------------------------------
  // This wave's blocks of tile j (DMA KiB i of the wave: KiB 4 i + wave of the tile).
  struct Bids { int b[C::DMA]; };
  auto bids_of = [&](int j) __attribute__((always_inline)) {
    Bids x;
#pragma unroll
    for (int i = 0; i < C::DMA; ++i) x.b[i] = s_bid[first_block(j) + (i * kGroupWaves + wave) / kKib];
    return x;
  };
  auto uniform = [&](Bids x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < C::DMA; ++i) x.b[i] = __builtin_amdgcn_readfirstlane(x.b[i]);
    return x;
  };
  auto dma_one = [&](bool isv, int j, const Bids& x, int i) __attribute__((always_inline)) {
    unsigned char* dst = (isv ? v_raw : k_raw) + (j & 1) * C::RAW + wave * 1024;
    const uint8_t* pages = (isv ? c.v_pages : c.k_pages) + wave % kKib * 1024;
    const u32x4 rsrc = buffer_rsrc(pages + (static_cast<size_t>(static_cast<uint32_t>(max(x.b[i], 0))) * (kScaleRows * D)),
                                   x.b[i] >= 0 ? 1024 : 0);
    dma16_to_lds(rsrc, isv ? static_cast<int>(ul * 16) : k_off, dst + i * kGroupWaves * 1024);
  };
  auto dma = [&](bool isv, int j, const Bids& x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < C::DMA; ++i) dma_one(isv, j, x, i);
  };

  auto start = [&]() __attribute__((always_inline)) {
    const Bids x = uniform(bids_of(0));
    dma(false, 0, x);
    dma(true, 0, x);
    dma(false, 1, uniform(bids_of(1)));
  };

  // heavy items go out in order, the next round's in the reverse order
  auto item_at = [&](int round) __attribute__((always_inline)) {
    return round * a.lanes + (round & 1 ? a.lanes - 1 - wl : wl);
  };
  Item it;
  bool more = get_item<D>(a, item_at(0), &it);
  int seg_b = -1, seg_0 = 0, seg_1 = 0;     // the segment whose blocks are in LDS: key tiles,
  int seg_last = 0;                         // and the last block looked up (the tile may end in a later one)
  bool holes = false, primed = false;       // primed: its first DMAs are on the way
  for (int round = 1; more; ++round) {
    const int rows = it.n * a.group;
    if (THIN && rows - it.r0 <= kThinRows) {
      thin_item<D>(c, a, it, kvh, reinterpret_cast<float*>(s_dyn), &s_ml[0][0][0]);
      more = get_item<D>(a, item_at(round), &it);
      continue;
    }
    const int row = it.r0 + wave * 32 + l32;          // this lane's query row
    // rows past the request's are computed like its last and not stored
    const int tok = min(row, rows - 1) / a.group;
    const int lim = max(it.len - it.n + tok + 1, 0);  // keys the row attends
    // tiles from this one on hold keys that not all rows attend
    const int mask_from = max(it.len - it.n + it.r0 / a.group + 1, 0) / C::BN;
    const int blk_end = (tile_end(a, it) + kScaleRows - 1) / kScaleRows;

    // ---- state ---------------------------------------------------------------
    bf16x8_t q[C::STEPS - C::QL];
    {
      const bf16* src = a.q + static_cast<size_t>(it.q0 + tok) * a.q_stride +
                        static_cast<size_t>(kvh * a.group + min(row, rows - 1) - tok * a.group) * D + 8 * hf;
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        const u32x4 w = ld16(src + 16 * s);
        if (s >= C::QL) q[s - C::QL] = as_bf16x8(w);
        else if (grp == 0) *reinterpret_cast<u32x4*>(s_q + ((wave * C::QL + s) * 64 + lane) * 16) = w;   // read behind barriers
      }
    }
    f32x16 o[C::DT], sc[C::KT];
    u32x4 p[C::KT][2];
#pragma unroll
    for (int d = 0; d < C::DT; ++d) o[d] = f32x16{};
    float m = -INFINITY, l = 0.f;

    if (it.t0 == it.t1) {     // no keys: straight to the output
      __syncthreads();
      if (threadIdx.x == 0) s_any_nan = 0;
    }
    for (int s0 = it.t0; s0 < it.t1; s0 += C::SEG / C::NB - 8) {
      const int s1 = min(it.t1, s0 + C::SEG / C::NB - 8);
      const int count = (s1 - s0 + 1) / 2;         // tiles of a group, the last of group 1 perhaps none
      const int last = min(blk_end, s1 * C::NB), fill = (2 * count + 8) * C::NB;
      const bool reuse = seg_b == it.b && seg_0 == s0 && s1 <= seg_1 && last <= seg_last && s1 == it.t1 && it.rec < 0;
      if (!reuse) {
        bool hole = false;
        for (int i = threadIdx.x; i < fill; i += kThreads) {
          const int blk = s0 * C::NB + i;
          const int bid = blk < last ? block_id(c, it.b, kvh, blk) : -1;
          hole |= blk < last && bid < 0;
          s_bid[i] = bid;
        }
        holes = __syncthreads_or(hole);
        seg_b = it.b;
        seg_0 = s0;
        seg_1 = s1;
        seg_last = last;
      }

      // ---- codes -> operands ----------------------------------------------
      // K: a thread takes KI 16-code pieces of one row, kStep apart.
      constexpr int kStep = kGroup / C::BN;
      struct RawK { u32x4 w[C::KI]; float sc; };
      auto load_k = [&](int j) __attribute__((always_inline)) {
        RawK x;
        const unsigned char* raw = k_raw + (j & 1) * C::RAW;
#pragma unroll
        for (int i = 0; i < C::KI; ++i) x.w[i] = ld16(raw + (kStep < 8 ? k_from ^ (i * kStep * 16) : k_from + i * kStep * 16));
        x.sc = s_ks[first_block(j) + cr / kScaleRows];
        return x;
      };
      auto store_k = [&](const RawK& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2 * C::KI; ++i) {
          const uint32_t lo = x.w[i >> 1][2 * (i & 1)], hi = x.w[i >> 1][2 * (i & 1) + 1];
          *reinterpret_cast<u32x4*>(k_ops + k_to + (i >> 1) * kStep * 1024 + (i & 1) * 512) =
              u32x4{fp8x2_to_bf16x2<false>(lo, x.sc), fp8x2_to_bf16x2<true>(lo, x.sc), fp8x2_to_bf16x2<false>(hi, x.sc),
                    fp8x2_to_bf16x2<true>(hi, x.sc)};
        }
      };
      // V: a thread takes 8 keys x 4 dims, the keys 16 (oc / 2) + 4 (oc % 2) + {0..3, 8..11}.
      struct RawV { uint32_t v[8]; float sc; };
      auto load_v = [&](int j) __attribute__((always_inline)) {
        RawV x;
        const unsigned char* raw = v_raw + (j & 1) * C::RAW + v_from;
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] = *reinterpret_cast<const uint32_t*>(raw + ((e & 3) + 8 * (e >> 2)) * D);
        x.sc = s_vs[first_block(j) + (oc >> 1)];
        return x;
      };
      // 0 times NaN is NaN: a masked row must not carry one into the product. NaN
      // codes are taken out and remembered by dim; the epilogue puts NaN into the
      // rows that attend the first.
      auto clean_v = [&](RawV& x, int j) __attribute__((always_inline)) {
        const uint32_t keep = s_bid[first_block(j) + (oc >> 1)] >= 0 ? 0xffffffffu : 0u;
        uint32_t seen = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t n = nan_codes(x.v[e]) >> 7;
          seen |= n & keep;
          x.v[e] &= keep & ~(n * 0xffu);
        }
        if (seen) {
          const unsigned char* raw = v_raw + (j & 1) * C::RAW + v_from;
          const int key = s0 * C::BN + first_block(j) * kScaleRows + 16 * (oc >> 1) + 4 * (oc & 1);
#pragma unroll 1
          for (int e = 0; e < 32; ++e) {
            const int r = (e >> 2 & 3) + 8 * (e >> 4);
            if ((raw[r * D + (e & 3)] & 0x7f) == 0x7f) {
              s_any_nan = 1;
              atomicMin(&s_nan[4 * dq + (e & 3)], key + r);
            }
          }
        }
      };
      auto store_v = [&](const RawV& x) __attribute__((always_inline)) {
        u32x4 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = __builtin_amdgcn_perm(x.v[2 * e + 1], x.v[2 * e], 0x05010400u);
          const uint32_t hi = __builtin_amdgcn_perm(x.v[2 * e + 1], x.v[2 * e], 0x07030602u);
          w[0][e] = fp8x2_to_bf16x2<false>(lo, x.sc);
          w[1][e] = fp8x2_to_bf16x2<true>(lo, x.sc);
          w[2][e] = fp8x2_to_bf16x2<false>(hi, x.sc);
          w[3][e] = fp8x2_to_bf16x2<true>(hi, x.sc);
        }
        // dim i of the quad: the next part, or for D = 64 the other half of this one
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x4*>(v_ops + v_to + (D == 64 ? (i >> 1) * 1024 + (i & 1) * 256 : i * 1024)) = w[i];
      };
      const bool v_threads = D != 64 || wave < 2;     // whole waves

      // ---- products ----------------------------------------------------------
      // A matrix phase: O += V P of the tile before (PV), then S = K Q of this one
      // (QK), one row of products whose operands are read AHEAD ahead of them. What
      // else the phase has to do (the next DMAs) goes between the products, a step
      // every second one, where it costs no time; the schedule barriers keep it all
      // so (left alone, the compiler reads the operands first, and spills).
      constexpr int NP = 2 * C::KT * C::DT, NQ = C::KT * C::STEPS;
      bf16x8_t ahead[C::AHEAD];     // the first operands of QK, read during PV
      auto load_qk = [&](int i) __attribute__((always_inline)) {
        return as_bf16x8(ld16(k_ops + ((i % C::KT * C::STEPS + i / C::KT) * 64 + lane) * 16));
      };
      auto pv = [&](auto&& step) __attribute__((always_inline)) {
        auto load = [&](int i) __attribute__((always_inline)) { return as_bf16x8(ld16(v_ops + (i * 64 + lane) * 16)); };
        bf16x8_t x[NP];
#pragma unroll
        for (int i = 0; i < C::AHEAD; ++i) x[i] = load(i);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (i + C::AHEAD < NP) x[i + C::AHEAD] = load(i + C::AHEAD);
          else ahead[i + C::AHEAD - NP] = load_qk(i + C::AHEAD - NP);
          const int s = i / C::DT, d = i % C::DT;
          o[d] = mfma32(x[i], as_bf16x8(p[s >> 1][s & 1]), o[d]);
          if (i & 1) step(i / 2);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto scores = [&]() __attribute__((always_inline)) {
        bf16x8_t x[NQ];
#pragma unroll
        for (int i = 0; i < C::AHEAD; ++i) x[i] = ahead[i];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          if (i + C::AHEAD < NQ) x[i + C::AHEAD] = load_qk(i + C::AHEAD);
          const int st = i / C::KT;
          const bf16x8_t qs = st >= C::QL ? q[st >= C::QL ? st - C::QL : 0]
                                          : as_bf16x8(ld16(s_q + ((wave * C::QL + st) * 64 + lane) * 16));
          sc[i % C::KT] = mfma32(x[i], qs, i < C::KT ? f32x16{} : sc[i % C::KT]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto softmax = [&](int j, bool masked) __attribute__((always_inline)) {
        if (masked) {
          const int rel = lim - s0 * C::BN - first_block(j) * kScaleRows - 4 * hf;
#pragma unroll
          for (int k = 0; k < C::KT; ++k) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int rb = s_bid[first_block(j) + 2 * k + g] >= 0 ? rel : -1;
#pragma unroll
              for (int i = 8 * g; i < 8 * g + 8; ++i)
                if (32 * k + 8 * (i >> 2) + (i & 3) >= rb) sc[k][i] = -INFINITY;
            }
          }
        }
        float t0 = sc[0][0], t1 = sc[0][8];     // two chains
#pragma unroll
        for (int k = 0; k < C::KT; ++k) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            t0 = fmaxf(t0, sc[k][i]);
            t1 = fmaxf(t1, sc[k][8 + i]);
          }
        }
        const float top = half_max(fmaxf(t0, t1)) * a.scale_log2;
        if (__ballot(top > m + kLazyLog2)) {
          const float mn = fmaxf(m, top);
          const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
          m = mn;
          l *= alpha;
#pragma unroll
          for (int d = 0; d < C::DT; ++d) o[d] *= alpha;
        }
        const float nm = m == -INFINITY ? 0.f : -m;
        float l1 = 0.f;
#pragma unroll
        for (int k = 0; k < C::KT; ++k) {
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = fast_exp2(fmaf(sc[k][i], a.scale_log2, nm));
          // P is rounded to bf16 once (half a step, 2^-8 of each weight, at random): its
          // sum of two, as the decode takes, would double this product. The sum is
          // taken of the rounded weights, in fp32, so that they add up to 1.
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[k][0][i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
            p[k][1][i] = pack_bf16x2(x[8 + 2 * i], x[9 + 2 * i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            l = add_pair(p[k][0][i], l);
            l1 = add_pair(p[k][1][i], l1);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) pin(p[k][i]);    // made in this phase, not where the next one uses it
        }
        l += l1;
      };
      const int mask_at = min(mask_from, s1);
      auto masked_tile = [&](int j) __attribute__((always_inline)) { return holes || s0 + 2 * j + grp >= mask_at; };

      // ---- the walk -------------------------------------------------------------
      if (!primed) start();
      if (!reuse) {
        for (int i = threadIdx.x; i < fill; i += kThreads) {
          const int bid = s_bid[i];
          s_ks[i] = bid >= 0 ? c.k_scale[bid] : 0.f;
          s_vs[i] = bid >= 0 ? c.v_scale[bid] : 0.f;
        }
      }
      primed = false;
      Bids bv, bk = uniform(bids_of(1));
      __builtin_amdgcn_s_waitcnt(vmcnt_imm<0>());
      __syncthreads();
      if (threadIdx.x < D && s0 == it.t0) s_nan[threadIdx.x] = kNoKey;
      if (threadIdx.x == 0 && s0 == it.t0) s_any_nan = 0;
      store_k(load_k(0));
      Bids next = bids_of(2);      // blocks of the tile whose K goes out next
      __syncthreads();
      if (grp == 1) phase_barrier();
      // In M(j): V of tile j + 1 and K of j + 2 (past the last tile: empty blocks).
      auto issue = [&](int j, int step) __attribute__((always_inline)) {
        if (step == 0) {
          bv = bk;
          bk = uniform(next);
        } else if (step <= C::DMA) {
          dma_one(true, j + 1, bv, step - 1);
        } else if (step <= 2 * C::DMA) {
          dma_one(false, j + 2, bk, step - 1 - C::DMA);
        } else if (step == 2 * C::DMA + 1) {
          next = bids_of(j + 3);
        }
      };
#pragma unroll
      for (int step = 0; step < 2 * C::DMA + 2; ++step) issue(0, step);
#pragma unroll
      for (int i = 0; i < C::AHEAD; ++i) ahead[i] = load_qk(i);
      scores();
      for (int j = 0;;) {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm<2 * C::DMA>());   // all but this phase's DMAs
        phase_barrier();
        // V(j): reads its codes, then softmax, then the operands change. (Converting
        // between the products of the matrix phase instead took as long: the vector
        // ALU, which both waves of a SIMD share, is what a phase waits for.)
        __builtin_amdgcn_s_setprio(0);
        const bool masked = masked_tile(j);
        const RawK rk = load_k(j + 1);
        RawV rv;
        if (v_threads) rv = load_v(j);
        softmax(j, masked);
        store_k(rk);
        if (v_threads) {
          if (masked) clean_v(rv, j);
          store_v(rv);
        }
        phase_barrier();
        // M(j + 1)
        __builtin_amdgcn_s_setprio(1);
        ++j;
        pv([&](int step) __attribute__((always_inline)) { issue(j, step); });
        if (j == count) break;
        scores();
      }
      if (grp == 0) phase_barrier();
      __builtin_amdgcn_s_waitcnt(vmcnt_imm<0>());
      __syncthreads();
    }

    // ---- the groups' states meet -----------------------------------------------
    // The next item's first codes are fetched meanwhile, if it walks the same keys.
    const Item done = it;
    more = get_item<D>(a, item_at(round), &it);
    if (more && it.b == seg_b && it.t0 == seg_0 && it.t0 < it.t1 && it.t1 <= seg_1 && it.rec < 0 &&
        (tile_end(a, it) + kScaleRows - 1) / kScaleRows <= seg_last && !(THIN && it.n * a.group - it.r0 <= kThinRows)) {
      start();
      primed = true;
    }
    l = half_sum(l);
    const int ln = here(threadIdx.x & 63), row32 = wave * 32 + (ln & 31);
    if (ln < 32) {
      s_ml[grp][row32][0] = m;
      s_ml[grp][row32][1] = l;
    }
    // Each group finishes half of the output: quads (4 rows of a part) {0, 1} and
    // {2, 3}, or, for D = 64, {0, 2} and {1, 3}; the other half it hands over.
    auto finish = [&](auto gtag) __attribute__((always_inline)) {
      constexpr int G = decltype(gtag)::value;
      constexpr int P = C::DT / C::XR;
      constexpr int kOwn[2] = {D == 64 ? G : 2 * G, D == 64 ? G + 2 : 2 * G + 1};
      constexpr int kOther[2] = {D == 64 ? 1 - G : 2 - 2 * G, D == 64 ? 3 - G : 3 - 2 * G};
      unsigned char* give = s_dyn + G * 2 * C::OPS + wave * P * 2048 + ln * 16;
      const unsigned char* take = s_dyn + (1 - G) * 2 * C::OPS + wave * P * 2048 + ln * 16;
      float f1 = 0.f, f2 = 0.f, mm = 0.f, ll = 0.f;
#pragma unroll
      for (int r = 0; r < C::XR; ++r) {
        if (r > 0) __syncthreads();
#pragma unroll
        for (int d = 0; d < P; ++d) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x16& x = o[r * P + d];
            *reinterpret_cast<f32x4*>(give + (d * 2 + i) * 1024) =
                f32x4{x[4 * kOther[i]], x[4 * kOther[i] + 1], x[4 * kOther[i] + 2], x[4 * kOther[i] + 3]};
          }
        }
        __syncthreads();
        if (r == 0) {
          const float m2 = s_ml[1 - G][row32][0], l2 = s_ml[1 - G][row32][1];
          mm = fmaxf(m, m2);
          f1 = m == -INFINITY ? 0.f : fast_exp2(m - mm);
          f2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - mm);
          ll = f1 * l + f2 * l2;
          if (done.rec < 0) {
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
            f1 *= inv;
            f2 *= inv;
          }
        }
#pragma unroll
        for (int d = 0; d < P; ++d) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(take + (d * 2 + i) * 1024);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = o[r * P + d][4 * kOwn[i] + e];
              o[r * P + d][4 * kOwn[i] + e] = y * f1 + x[e] * f2;
            }
          }
        }
      }
      const int hf = ln >> 5, row = done.r0 + row32;
      if (s_any_nan) {
        const int tok = row / a.group;
        const int lim = max(done.len - done.n + tok + 1, 0);
#pragma unroll
        for (int d = 0; d < C::DT; ++d) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (s_nan[out_dim<D>(d, 8 * kOwn[i] + 4 * hf + e)] < lim) o[d][4 * kOwn[i] + e] = __uint_as_float(0x7fc00000u);
          }
        }
      }
      if (done.rec >= 0) {
        if (done.r0 + wave * 32 >= done.n * a.group) return;     // no rows: not read
        float* rec = a.part + (static_cast<size_t>(done.rec) * c.Hkv + kvh) * C::REC;
#pragma unroll
        for (int d = 0; d < C::DT; ++d) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x16& x = o[d];
            *reinterpret_cast<f32x4*>(rec + (((wave * C::DT + d) * 4 + kOwn[i]) * 64 + ln) * 4) =
                f32x4{x[4 * kOwn[i]], x[4 * kOwn[i] + 1], x[4 * kOwn[i] + 2], x[4 * kOwn[i] + 3]};
          }
        }
        if (G == 0 && hf == 0) {
          rec[kRows * D + row32 * 2] = mm;
          rec[kRows * D + row32 * 2 + 1] = ll;
        }
      } else if (row < done.n * a.group) {
        const unsigned tok = static_cast<unsigned>(row) / static_cast<unsigned>(a.group);
        bf16* dst = a.out + (static_cast<size_t>(done.q0 + tok) * a.Hq + kvh * a.group + row - tok * a.group) * D;
        if constexpr (D == 64) {
#pragma unroll
          for (int e = 0; e < 4; ++e)   // dims 4 m + {0, 1, 2, 3} from rows m and m + 16 of both parts
            *reinterpret_cast<u32x2*>(dst + 4 * (8 * G + 4 * hf + e)) =
                u32x2{pack_bf16x2(o[0][4 * G + e], o[0][8 + 4 * G + e]), pack_bf16x2(o[1][4 * G + e], o[1][8 + 4 * G + e])};
        } else {
#pragma unroll
          for (int g = 0; g < D / 128; ++g) {
#pragma unroll
            for (int i = 8 * G; i < 8 * G + 8; ++i)
              *reinterpret_cast<u32x2*>(dst + 128 * g + 4 * (8 * (i >> 2) + 4 * hf + (i & 3))) =
                  u32x2{pack_bf16x2(o[4 * g][i], o[4 * g + 1][i]), pack_bf16x2(o[4 * g + 2][i], o[4 * g + 3][i])};
          }
        }
      }
    };
    if (grp == 0) finish(std::integral_constant<int, 0>{});
    else finish(std::integral_constant<int, 1>{});
  }
}

// Joins the records of a tile whose keys were cut: o = sum 2^(m_i - M) o_i /
// sum 2^(m_i - M) l_i. A workgroup takes 32 query rows and up to 128 dims; a
// thread's values are those of the main kernel's lane.
template <int D>
__global__ __launch_bounds__(256) void gqa_prefill_paged_fp8_merge_kernel(PagedFp8 c, Fp8PrefillArgs a) {
  using C = Cfg<D>;
  Item it;
  int rec, cuts;
  if (a.plan != nullptr) {
    if (static_cast<int>(blockIdx.x) >= a.plan[1]) return;
    const PlanCut x = reinterpret_cast<const PlanCut*>(reinterpret_cast<const PlanItem*>(a.plan + kPlanHead) +
                                                       plan_items(a.T, a.B, a.group, a.lanes))[blockIdx.x];
    load_request(a, x.b, &it);
    it.r0 = x.r0;
    rec = x.rec;
    cuts = x.cuts;
  } else {
    rec = static_cast<int>(blockIdx.x) * a.splits;
    cuts = a.splits;
    if (!get_item<D>(a, rec, &it)) return;
  }
  constexpr int G = D > 128 ? D / 128 : 1;
  const int kvh = blockIdx.y, wave = static_cast<int>(blockIdx.z) / G, g = static_cast<int>(blockIdx.z) % G;
  const int lane = threadIdx.x & 63, i = threadIdx.x >> 6, l32 = lane & 31, hf = lane >> 5;
  if (D == 64 && i > 1) return;
  const int row = it.r0 + wave * 32 + l32;
  if (row >= it.n * a.group) return;
  const size_t step = static_cast<size_t>(c.Hkv) * C::REC;
  const float* r0 = a.part + (static_cast<size_t>(rec) * c.Hkv + kvh) * C::REC;
  const float* ml = r0 + kRows * D + (wave * 32 + l32) * 2;
  // kBatch records at a time, their loads all in flight (past the last: the last
  // again, with weight 0).
  constexpr int kBatch = 4;
  float M = -INFINITY, L = 0.f;
  f32x4 o[4] = {};
  for (int x0 = 0; x0 < cuts; x0 += kBatch) {
    float m[kBatch], l[kBatch];
    f32x4 v[kBatch][4];
#pragma unroll
    for (int y = 0; y < kBatch; ++y) {
      const size_t at = min(x0 + y, cuts - 1) * step;
      m[y] = x0 + y < cuts ? ml[at] : -INFINITY;
      l[y] = ml[at + 1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dt = D == 64 ? e >> 1 : 4 * g + e, quad = D == 64 ? i + 2 * (e & 1) : i;
        v[y][e] = *reinterpret_cast<const f32x4*>(r0 + at + (((wave * C::DT + dt) * 4 + quad) * 64 + lane) * 4);
      }
    }
    float top = M;
#pragma unroll
    for (int y = 0; y < kBatch; ++y) top = fmaxf(top, m[y]);
    const float f0 = M == -INFINITY ? 0.f : fast_exp2(M - top);
    M = top;
    L *= f0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f0;
#pragma unroll
    for (int y = 0; y < kBatch; ++y) {
      if (x0 + y < cuts) {
        const float f = m[y] == -INFINITY ? 0.f : fast_exp2(m[y] - M);
        L += f * l[y];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += f * v[y][e];
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  bf16* dst = a.out + (static_cast<size_t>(it.q0 + row / a.group) * a.Hq + kvh * a.group + row % a.group) * D + 128 * g;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    *reinterpret_cast<u32x2*>(dst + 4 * (8 * i + 4 * hf + e)) =
        u32x2{pack_bf16x2(o[0][e] * inv, o[1][e] * inv), pack_bf16x2(o[2][e] * inv, o[3][e] * inv)};
}

// Workgroups per KV head, and key runs of one request's tiles: enough that all
// CUs have one, none shorter than kMinKeys where the length is the bound. As many
// runs for each tile, so a number of tiles a little above the workgroups', or above a
// half of them, leaves CUs without one (us, 16 / 4, D = 256 after 14000 rows, 64
// workgroups a head: 32 tiles 240, 33 367, 64 466, 65 757; 32 / 8, D = 128, 32
// workgroups: 32 tiles 242, 33 412).
void shape(int T, int B, int Hkv, int group, int max_len, int* lanes, int* splits) {
  const int tiles = static_cast<int>((static_cast<long>(T) * group + kRows - 1) / kRows);
  *lanes = std::max(1, kCus / Hkv);
  *splits = 1;
  if (B == 1 && tiles < *lanes) {
    const int runs = std::max(1, max_len / kMinKeys);
    *splits = std::min(*lanes / tiles, runs);
  }
}

template <int D>
size_t workspace_need(int T, int B, int Hkv, int group, int max_len, int* lanes, int* splits) {
  shape(T, B, Hkv, group, max_len, lanes, splits);
  const size_t rec = static_cast<size_t>(Cfg<D>::REC) * sizeof(float) * Hkv;
  if (B == 1) {
    const size_t tiles = (static_cast<size_t>(T) * group + kRows - 1) / kRows;
    return *splits > 1 ? tiles * *splits * rec : 0;
  }
  // runs of cut tiles: each tile has more than a share, and at most one run is left over
  return plan_bytes(T, B, group, *lanes) + 2 * static_cast<size_t>(*lanes) * rec;
}

template <int D>
int launch(PagedFp8 c, Fp8PrefillArgs a, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const size_t need = workspace_need<D>(a.T, a.B, c.Hkv, a.group, a.max_len, &a.lanes, &a.splits);
  const int tiles = static_cast<int>((static_cast<long>(a.T) * a.group + kRows - 1) / kRows);
  auto walk = [&](const PagedFp8& cache, const Fp8PrefillArgs& args) {
    // one request's last tile may be thin too, but is one of many then
    const bool thin = a.B > 1 || static_cast<long>(a.T) * a.group <= kThinRows;
    if (thin)
      hipLaunchKernelGGL((gqa_prefill_paged_fp8_kernel<D, true>), dim3(args.lanes * c.Hkv), dim3(kThreads), Cfg<D>::LDS, st, cache, args);
    else
      hipLaunchKernelGGL((gqa_prefill_paged_fp8_kernel<D, false>), dim3(args.lanes * c.Hkv), dim3(kThreads), Cfg<D>::LDS, st, cache, args);
  };
  auto merge = [&](int cut_tiles) {
    hipLaunchKernelGGL((gqa_prefill_paged_fp8_merge_kernel<D>), dim3(cut_tiles, c.Hkv, 4 * (D > 128 ? D / 128 : 1)), dim3(256), 0,
                       st, c, a);
  };
  if (a.B == 1) {
    if (workspace == nullptr || workspace_bytes < need) a.splits = 1;
    a.part = static_cast<float*>(workspace);
    a.lanes = static_cast<int>(std::min<long>(a.lanes, static_cast<long>(tiles) * a.splits));
    walk(c, a);
    if (a.splits > 1) merge(tiles);
  } else if (workspace == nullptr) {
    // one request after the other
    a.lanes = std::min(a.lanes, tiles);
    for (int b = 0; b < a.B; ++b) {
      walk(c, a);
      c.table += c.max_pages;
      ++a.query_start;
      ++a.seq_lens;
    }
  } else {
    if (workspace_bytes < need)
      return set_error(AILA_HIP_EWORKSPACE, "gqa_prefill_paged_fp8: a workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    a.plan = static_cast<int*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan_bytes(a.T, a.B, a.group, a.lanes));
    auto plan = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3(1), dim3(threads), static_cast<size_t>(3 * a.B + 1) * sizeof(int), st, a, Cfg<D>::BN);
    };
    // a thread a tile; few tiles: 4 waves, whose sums and barriers are shorter (us, a batch of
    // 32 with 91 tiles: 5.4 against 7.1)
    if (a.B <= 256 && plan_items(a.T, a.B, a.group, 0) <= 256) plan(gqa_prefill_paged_fp8_plan_kernel<256>, 256);
    else plan(gqa_prefill_paged_fp8_plan_kernel<1024>, 1024);
    walk(c, a);
    merge(a.lanes);
  }
  return check_launch("gqa_prefill_paged_fp8");
}

}  // namespace
}  // namespace aila

extern "C" size_t aila_hip_gqa_prefill_paged_fp8_workspace_size(int T, int B, int Hq, int Hkv, int D, int max_len) {
  using namespace aila;
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_len < 0) return 0;
  int lanes, splits;
  switch (D) {
    case 64: return workspace_need<64>(T, B, Hkv, Hq / Hkv, max_len, &lanes, &splits);
    case 128: return workspace_need<128>(T, B, Hkv, Hq / Hkv, max_len, &lanes, &splits);
    case 256: return workspace_need<256>(T, B, Hkv, Hq / Hkv, max_len, &lanes, &splits);
    default: return 0;
  }
}

extern "C" int aila_hip_gqa_prefill_paged_fp8(const void* q, long q_stride, const void* k_pages, const void* v_pages,
                                              const float* k_scale, const float* v_scale, void* out, void* workspace,
                                              size_t workspace_bytes, int T, int B, int Hq, int Hkv, int D,
                                              int page_size, int num_pages, const int* block_table, int max_pages,
                                              int max_len, const int* query_start, const int* seq_lens, void* stream) {
  using namespace aila;
  AILA_REQUIRE(q && out && block_table && query_start && seq_lens, "gqa_prefill_paged_fp8: null pointer");
  if (int rc = check_paged_fp8("gqa_prefill_paged_fp8", k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages))
    return rc;
  AILA_REQUIRE(B > 0 && B <= kMaxSequences, "gqa_prefill_paged_fp8: B=%d outside [1, %d]", B, kMaxSequences);
  AILA_REQUIRE(Hq > 0 && Hq % Hkv == 0 && Hq <= 65535, "gqa_prefill_paged_fp8: bad heads (Hq=%d Hkv=%d)", Hq, Hkv);
  AILA_REQUIRE(T > 0 && static_cast<long>(T) * (Hq / Hkv) <= (1L << 30), "gqa_prefill_paged_fp8: T=%d tokens are too many", T);
  AILA_REQUIRE(q_stride >= static_cast<long>(Hq) * D && q_stride % 8 == 0,
               "gqa_prefill_paged_fp8: query stride %ld must be a multiple of 8 and hold Hq * D = %ld values", q_stride,
               static_cast<long>(Hq) * D);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "gqa_prefill_paged_fp8: q, out and workspace must be 16-byte aligned");
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30),
               "gqa_prefill_paged_fp8: bad max_pages=%d", max_pages);
  AILA_REQUIRE(max_len >= 0 && max_len <= max_pages * page_size, "gqa_prefill_paged_fp8: max_len=%d outside [0, %d]",
               max_len, max_pages * page_size);
  PagedFp8 c{static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages), k_scale, v_scale,
             block_table, max_pages, num_pages, Hkv, page_size / kScaleRows};
  Fp8PrefillArgs a{};
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<bf16*>(out);
  a.query_start = query_start;
  a.seq_lens = seq_lens;
  a.T = T; a.B = B; a.Hq = Hq; a.group = Hq / Hkv;
  a.max_len = max_len;
  a.scale_log2 = kLog2e / sqrtf(static_cast<float>(D));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (D) {
    case 64: return launch<64>(c, a, workspace, workspace_bytes, st);
    case 128: return launch<128>(c, a, workspace, workspace_bytes, st);
    default: return launch<256>(c, a, workspace, workspace_bytes, st);
  }
}
