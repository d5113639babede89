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
// both fed, by one wave each.
#include "paged_fp8.hpp"

#include <algorithm>

namespace aila {
namespace {

constexpr int kGroupWaves = 4;
constexpr int kGroup = 64 * kGroupWaves;   // threads of a group
constexpr int kThreads = 2 * kGroup;
constexpr int kRows = 32 * kGroupWaves;    // query rows of a tile
constexpr int kMaxSequences = 4096;
constexpr int kCus = 256;
constexpr int kNoKey = 0x7fffffff;


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
  static constexpr int AHEAD = D == 256 ? 2 : 4;  // LDS operand reads in flight ahead of their MFMAs
  static constexpr int GROUP_LDS = 2 * OPS + 4 * RAW;
  static constexpr int LDS = 2 * GROUP_LDS;
  static_assert(LDS >= kGroupWaves * DT * 16 * 64 * 4, "the groups' outputs meet in LDS");
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
  const int rank = index / a.splits, cut = index % a.splits;
  if (rank >= tiles) return false;
  it->r0 = (tiles - 1 - rank) * kRows;
  const int kt = (tile_end(a, *it) + Cfg<D>::BN - 1) / Cfg<D>::BN;
  it->t0 = static_cast<int>(static_cast<long>(kt) * cut / a.splits);
  it->t1 = static_cast<int>(static_cast<long>(kt) * (cut + 1) / a.splits);
  it->rec = a.splits > 1 ? index : -1;
  return true;
}

// The items of a ragged batch. Each workgroup of a KV head should get the same
// number of key tiles: a tile of query rows with more of them than that share
// is cut into equal runs of at most a share, and the items are sorted by size,
// so that the workgroups, which take them forth and back, fill up evenly.
constexpr int kPlanThreads = 1024;
constexpr int kMinRun = 8;      // key tiles; shorter runs cost more in records than they gain
constexpr int kBuckets = 1024;

template <typename T>
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
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += s_wave[w];
    all += s_wave[w];
  }
  *total = all;
  return x + before;   // inclusive
}

__global__ __launch_bounds__(kPlanThreads) void gqa_prefill_paged_fp8_plan_kernel(Fp8PrefillArgs a, int key_tile) {
  extern __shared__ int s_first[];     // [B + 1] first tile of each request
  __shared__ int s_wave[kPlanThreads / 64];
  __shared__ long s_wave_l[kPlanThreads / 64];
  __shared__ int s_bucket[kBuckets];
  __shared__ unsigned long long s_sum;
  const int tid = threadIdx.x;
  PlanItem* items = reinterpret_cast<PlanItem*>(a.plan + kPlanHead);
  PlanCut* cuts_of = reinterpret_cast<PlanCut*>(items + plan_items(a.T, a.B, a.group, a.lanes));
  s_bucket[tid] = 0;
  if (tid == 0) {
    s_first[0] = 0;
    s_sum = 0;
  }
  // malformed starts may overlap: no more tiles than the list holds
  const long most = plan_items(a.T, a.B, a.group, 0);
  long all_tiles = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    Item it{};
    if (b < a.B) load_request(a, b, &it);
    long all;
    const long incl = all_tiles + plan_scan<long>((it.n * a.group + kRows - 1) / kRows, s_wave_l, &all);
    if (b < a.B) s_first[b + 1] = static_cast<int>(min(incl, most));
    all_tiles += all;
  }
  const int tiles = static_cast<int>(min(all_tiles, most));
  __syncthreads();
  auto tile = [&](int f, Item* it) __attribute__((always_inline)) {   // -> key tiles
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_first[mid] <= f) lo = mid; else hi = mid;
    }
    load_request(a, lo, it);
    it->r0 = (f - s_first[lo]) * kRows;
    return (tile_end(a, *it) + key_tile - 1) / key_tile;
  };
  unsigned long long sum = 0;
  for (int f = tid; f < tiles; f += kPlanThreads) {
    Item it;
    sum += tile(f, &it);
  }
  atomicAdd(&s_sum, sum);
  __syncthreads();
  const int share = max(kMinRun, static_cast<int>((s_sum + a.lanes - 1) / a.lanes));
  auto bucket = [&](int size) __attribute__((always_inline)) {   // large sizes first
    return kBuckets - 1 - static_cast<int>(static_cast<long>(size) * (kBuckets - 1) / share);
  };
  for (int f = tid; f < tiles; f += kPlanThreads) {
    Item it;
    const int kt = tile(f, &it), cuts = max(1, (kt + share - 1) / share);
    for (int i = 0; i < cuts; ++i)
      atomicAdd(&s_bucket[bucket(static_cast<int>(static_cast<long>(kt) * (i + 1) / cuts - static_cast<long>(kt) * i / cuts))], 1);
  }
  __syncthreads();
  const int mine = s_bucket[tid];
  int total;
  const int incl = plan_scan<int>(mine, s_wave, &total);
  s_bucket[tid] = incl - mine;
  __syncthreads();
  // Which workgroup an item goes to depends on the order within a bucket, its
  // result does not: records are numbered by the tiles' order.
  int recs = 0, cut_tiles = 0;
  for (int f0 = 0; f0 < tiles; f0 += kPlanThreads) {
    const int f = f0 + tid;
    Item it{};
    int kt = 0, cuts = 0;
    if (f < tiles) {
      kt = tile(f, &it);
      cuts = max(1, (kt + share - 1) / share);
    }
    const int cut = cuts > 1;
    int all_r, all_c;
    const int rec = recs + plan_scan<int>(cut ? cuts : 0, s_wave, &all_r) - (cut ? cuts : 0);
    const int slot = cut_tiles + plan_scan<int>(cut, s_wave, &all_c) - cut;
    recs += all_r;
    cut_tiles += all_c;
    if (cut) cuts_of[slot] = PlanCut{it.b, it.r0, rec, cuts};
    for (int i = 0; i < cuts; ++i) {
      const int t0 = static_cast<int>(static_cast<long>(kt) * i / cuts), t1 = static_cast<int>(static_cast<long>(kt) * (i + 1) / cuts);
      items[atomicAdd(&s_bucket[bucket(t1 - t0)], 1)] = PlanItem{it.b, it.r0, t0, t1, cut ? rec + i : -1};
    }
  }
  if (tid == 0) {
    a.plan[0] = total;
    a.plan[1] = cut_tiles;
  }
}

template <int D>
__global__ __launch_bounds__(kThreads, 1) void gqa_prefill_paged_fp8_kernel(PagedFp8 c, Fp8PrefillArgs a) {
  using C = Cfg<D>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char s_dyn[];
  __shared__ int s_nan[D];      // first masked-tile key whose V holds NaN in this dim
  __shared__ float s_ml[kRows][2];
  const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / kGroup);
  const int t = threadIdx.x % kGroup, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  unsigned char* mine = s_dyn + grp * C::GROUP_LDS;
  unsigned char* k_ops = mine;
  unsigned char* v_ops = mine + C::OPS;
  unsigned char* k_raw = mine + 2 * C::OPS;            // two tiles
  unsigned char* v_raw = k_raw + 2 * C::RAW;           // two tiles
  const int kvh = static_cast<int>(blockIdx.x) % c.Hkv, wl = static_cast<int>(blockIdx.x) / c.Hkv;

  for (int round = 0;; ++round) {
    // heavy items go out in order, the next round's in the reverse order
    const int index = round * a.lanes + (round & 1 ? a.lanes - 1 - wl : wl);
    Item it;
    if (!get_item<D>(a, index, &it)) break;   // nor is there a later one
    const int rows = it.n * a.group;
    const int row = it.r0 + wave * 32 + l32;          // this lane's query row
    const bool there = row < rows;
    const int tok = there ? row / a.group : 0;
    const int h = kvh * a.group + row % a.group;
    const int lim = there ? max(it.len - it.n + tok + 1, 0) : 0;    // keys it attends
    const int full = max(it.len - it.n + it.r0 / a.group + 1, 0);   // keys that all rows attend
    const int end = max(it.len - it.n + min(it.n - 1, (it.r0 + kRows - 1) / a.group) + 1, 0);
    const bool ragged = it.r0 + kRows > rows;
    const int blk_end = (end + kScaleRows - 1) / kScaleRows;
    const int count = (it.t1 - it.t0 + 1) / 2;         // tiles of a group, the last of group 1 perhaps none
    auto tile_of = [&](int j) __attribute__((always_inline)) { return it.t0 + 2 * j + grp; };

    if (threadIdx.x < D) s_nan[threadIdx.x] = kNoKey;

    // Blocks of 1024 keys at a time, lane i the i-th: the current ones and the next.
    constexpr int kTilesPerRef = 1024 / C::BN;
    int ref_at = tile_of(0) / kTilesPerRef;
    auto fetch = [&](int at) __attribute__((always_inline)) { return block_ref(c, it.b, kvh, at * 64 + lane, blk_end); };
    BlockRef ra = fetch(ref_at), rb = fetch(ref_at + 1);
    auto advance = [&](int tile) __attribute__((always_inline)) {
      if (tile / kTilesPerRef > ref_at) {
        ++ref_at;
        ra = rb;
        rb = fetch(ref_at + 1);
      }
    };
    // block `i` (0 .. NB-1) of a tile
    auto ref_lane = [&](int tile, int i) __attribute__((always_inline)) { return (tile * C::NB + i) & 63; };
    auto bid_of = [&](int tile, int i) __attribute__((always_inline)) {
      const int x = tile / kTilesPerRef > ref_at ? rb.bid : ra.bid;
      const int bid = __builtin_amdgcn_readlane(x, ref_lane(tile, i));
      return tile < it.t1 ? bid : -1;
    };

    // ---- DMA of a tile's codes -------------------------------------------
    auto dma = [&](bool isv, int j) __attribute__((always_inline)) {
      const int tile = tile_of(j);
      unsigned char* dst = (isv ? v_raw : k_raw) + (j & 1) * C::RAW;
      const uint8_t* pages = isv ? c.v_pages : c.k_pages;
      const int ln = here(lane);
#pragma unroll
      for (int i = 0; i < C::DMA; ++i) {
        const int piece = i * kGroupWaves + wave;               // KiB of the tile
        const int bid = bid_of(tile, piece * 1024 / (kScaleRows * D));
        const u32x4 rsrc = buffer_rsrc(pages + static_cast<size_t>(max(bid, 0)) * (kScaleRows * D), bid >= 0 ? kScaleRows * D : 0);
        const int idx = piece * 64 + ln;
        const int r = idx / C::CH, p = idx % C::CH;
        const int off = (r % kScaleRows) * D + (isv ? p : p ^ piece_swizzle<D>(r)) * 16;
        dma16_to_lds(rsrc, off, dst + piece * 1024);
      }
    };

    // ---- codes -> operands ------------------------------------------------
    auto scale_of = [&](bool isv, int tile, int blk) __attribute__((always_inline)) {
      const bool next = tile / kTilesPerRef > ref_at;
      return __shfl(isv ? (next ? rb.vs : ra.vs) : (next ? rb.ks : ra.ks), ref_lane(tile, blk));
    };
    auto convert_k = [&](int j) __attribute__((always_inline)) {
      const int th = here(t);
      const int r = th % C::BN, s0 = th / C::BN;
      constexpr int kStep = kGroup / C::BN;
      const float sc = scale_of(false, tile_of(j), r / kScaleRows);
      unsigned char* dst0 = k_ops + (((r / 32) * C::STEPS + s0) * 64 + (r & 31)) * 16;
      const unsigned char* raw0 = k_raw + (j & 1) * C::RAW + r * D;
#pragma unroll
      for (int i = 0; i < C::KI; ++i) {
        const int s = s0 + kStep * i;                            // piece: MFMA step s
        const u32x4 w = ld16(raw0 + ((s ^ piece_swizzle<D>(r)) << 4));
        unsigned char* dst = dst0 + kStep * i * 1024;
        *reinterpret_cast<u32x4*>(dst) = u32x4{fp8x2_to_bf16x2<false>(w[0], sc), fp8x2_to_bf16x2<true>(w[0], sc),
                                               fp8x2_to_bf16x2<false>(w[1], sc), fp8x2_to_bf16x2<true>(w[1], sc)};
        *reinterpret_cast<u32x4*>(dst + 512) = u32x4{fp8x2_to_bf16x2<false>(w[2], sc), fp8x2_to_bf16x2<true>(w[2], sc),
                                                     fp8x2_to_bf16x2<false>(w[3], sc), fp8x2_to_bf16x2<true>(w[3], sc)};
      }
    };
    // bit i: block i of the tile has a page and is this run's
    constexpr unsigned kAllBlocks = (1u << C::NB) - 1;
    auto held_blocks = [&](int tile) __attribute__((always_inline)) {
      const int x = tile / kTilesPerRef > ref_at ? rb.bid : ra.bid;
      return tile < it.t1 ? static_cast<unsigned>(__ballot(x >= 0) >> ref_lane(tile, 0)) & kAllBlocks : 0u;
    };
    auto is_masked = [&](int tile) __attribute__((always_inline)) {
      return ragged || (tile + 1) * C::BN > full || held_blocks(tile) != kAllBlocks;
    };
    auto convert_v = [&](int j) __attribute__((always_inline)) {
      if (D == 64 && wave >= 2) return;
      const unsigned char* raw = v_raw + (j & 1) * C::RAW;
      const int th = here(t);
      const int o = th / (D / 4), dq = th % (D / 4);             // 8 keys x 4 dims
      const int st = o >> 1, h8 = o & 1;                         // 16-key step of the tile, half
      const int key = 16 * st + 4 * h8;
      const float sc = scale_of(true, tile_of(j), st);
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = *reinterpret_cast<const uint32_t*>(raw + (key + (e & 3) + 8 * (e >> 2)) * D + 4 * dq);
      if (is_masked(tile_of(j))) {
        if (!(held_blocks(tile_of(j)) >> st & 1)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0u;
        }
        // 0 times NaN is NaN: a masked row must not carry one into the product.
        // NaN codes are taken out and remembered by dim; the epilogue puts NaN
        // into the rows that attend the first.
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t n = nan_codes(v[e]);
          if (n) {
            v[e] &= ~((n >> 7) * 0xffu);
            for (; n; n &= n - 1)
              atomicMin(&s_nan[4 * dq + (__builtin_ctz(n) >> 3)], tile_of(j) * C::BN + key + (e & 3) + 8 * (e >> 2));
          }
        }
      }
      u32x4 w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = __builtin_amdgcn_perm(v[2 * e + 1], v[2 * e], 0x05010400u);
        const uint32_t hi = __builtin_amdgcn_perm(v[2 * e + 1], v[2 * e], 0x07030602u);
        w[0][e] = fp8x2_to_bf16x2<false>(lo, sc);
        w[1][e] = fp8x2_to_bf16x2<true>(lo, sc);
        w[2][e] = fp8x2_to_bf16x2<false>(hi, sc);
        w[3][e] = fp8x2_to_bf16x2<true>(hi, sc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int dt, m;
        out_slot<D>(dq, i, &dt, &m);
        *reinterpret_cast<u32x4*>(v_ops + ((st * C::DT + dt) * 64 + h8 * 32 + m) * 16) = w[i];
      }
    };

    // ---- state ---------------------------------------------------------------
    bf16x8_t q[C::STEPS];
#pragma unroll
    for (int s = 0; s < C::STEPS; ++s) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if (there) w = ld16(a.q + static_cast<size_t>(it.q0 + tok) * a.q_stride + static_cast<size_t>(h) * D + 16 * s + 8 * hf);
      q[s] = as_bf16x8(w);
    }
    f32x16 o[C::DT], sc[C::KT];
    u32x4 p[C::KT][2];
#pragma unroll
    for (int d = 0; d < C::DT; ++d) o[d] = f32x16{};
    float m = -INFINITY, l = 0.f;

    // Operands are read AHEAD ahead of the products that take them; the schedule
    // barriers keep it so (left alone, the compiler reads them all first, and
    // spills).
    auto pv = [&]() __attribute__((always_inline)) {
      constexpr int N = 2 * C::KT * C::DT;
      bf16x8_t v[N];
#pragma unroll
      for (int i = 0; i < C::AHEAD && i < N; ++i) v[i] = as_bf16x8(ld16(v_ops + (i * 64 + lane) * 16));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + C::AHEAD < N) v[i + C::AHEAD] = as_bf16x8(ld16(v_ops + ((i + C::AHEAD) * 64 + lane) * 16));
        const int s = i / C::DT, d = i % C::DT;
        o[d] = mfma32(v[i], as_bf16x8(p[s >> 1][s & 1]), o[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto scores = [&]() __attribute__((always_inline)) {
      constexpr int N = C::KT * C::STEPS;
      auto load = [&](int i) __attribute__((always_inline)) {
        return as_bf16x8(ld16(k_ops + ((i % C::KT * C::STEPS + i / C::KT) * 64 + lane) * 16));
      };
      bf16x8_t k[N];
#pragma unroll
      for (int x = 0; x < C::KT; ++x) sc[x] = f32x16{};
#pragma unroll
      for (int i = 0; i < C::AHEAD && i < N; ++i) k[i] = load(i);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + C::AHEAD < N) k[i + C::AHEAD] = load(i + C::AHEAD);
        sc[i % C::KT] = mfma32(k[i], q[i / C::KT], sc[i % C::KT]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto softmax = [&](int j) __attribute__((always_inline)) {
      const int tile = tile_of(j);
      if (is_masked(tile)) {
        const unsigned held = held_blocks(tile);
        const int rel = lim - tile * C::BN - 4 * hf;
#pragma unroll
        for (int k = 0; k < C::KT; ++k) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool ok = held >> (2 * k + (i >> 3)) & 1;
            if (!(ok && 32 * k + 8 * (i >> 2) + (i & 3) < rel)) sc[k][i] = -INFINITY;
          }
        }
      }
      float top = sc[0][0];
#pragma unroll
      for (int k = 0; k < C::KT; ++k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[k][i]);
      }
      top = half_max(top) * a.scale_log2;
      if (__ballot(top > m + kLazyLog2)) {
        const float mn = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < C::DT; ++d) o[d] *= alpha;
      }
      const float nm = m == -INFINITY ? 0.f : -m;
#pragma unroll
      for (int k = 0; k < C::KT; ++k) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] = fast_exp2(fmaf(sc[k][i], a.scale_log2, nm));
          l += x[i];
        }
        // P is rounded to bf16 once (2^-9 of each weight, at random): its sum of two,
        // as the decode takes, would double this product.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[k][0][i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
          p[k][1][i] = pack_bf16x2(x[8 + 2 * i], x[9 + 2 * i]);
        }
      }
    };

    // ---- the walk ---------------------------------------------------------------
    dma(false, 0);
    dma(true, 0);
    dma(false, 1);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm<0>());
    __syncthreads();
    convert_k(0);
    __syncthreads();
    if (grp == 1) phase_barrier();
    for (int j = 0; j <= count; ++j) {
      // M(j)
      if (j < count) {
        dma(false, j + 2);
        dma(true, j + 1);
      }
      if (j > 0) pv();
      if (j < count) scores();
      __builtin_amdgcn_s_waitcnt(vmcnt_imm<2 * C::DMA>());   // all but this phase's DMAs
      phase_barrier();
      // V(j)
      if (j < count) {
        advance(tile_of(j));
        convert_v(j);
        __builtin_amdgcn_sched_barrier(0);
        convert_k(j + 1);
        __builtin_amdgcn_sched_barrier(0);
        softmax(j);
      }
      phase_barrier();
    }
    if (grp == 0) phase_barrier();
    __builtin_amdgcn_s_waitcnt(vmcnt_imm<0>());
    __syncthreads();

    // ---- the groups' states meet ---------------------------------------------
    {
    const int lane = here(threadIdx.x & 63), l32 = lane & 31, hf = lane >> 5;
    const int row = it.r0 + wave * 32 + l32;
    const bool there = row < rows;
    const int tok = there ? row / a.group : 0;
    const int h = kvh * a.group + row % a.group;
    l = half_sum(l);
    float* s_o = reinterpret_cast<float*>(s_dyn);                                    // [wave][part][quad][lane] f32x4
    if (grp == 1) {
#pragma unroll
      for (int d = 0; d < C::DT; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(s_o + (((wave * C::DT + d) * 4 + i) * 64 + lane) * 4) =
              f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      }
      if (hf == 0) {
        s_ml[wave * 32 + l32][0] = m;
        s_ml[wave * 32 + l32][1] = l;
      }
    }
    __syncthreads();
    if (grp == 0) {
      const float m2 = s_ml[wave * 32 + l32][0], l2 = s_ml[wave * 32 + l32][1];
      const float mm = fmaxf(m, m2);
      const float f1 = m == -INFINITY ? 0.f : fast_exp2(m - mm), f2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - mm);
      const float ll = f1 * l + f2 * l2;
      const float inv = it.rec >= 0 ? 1.0f : ll == 0.f ? 0.f : 1.0f / ll;
      float* rec = it.rec >= 0 ? a.part + (static_cast<size_t>(it.rec) * c.Hkv + kvh) * C::REC : nullptr;
#pragma unroll
      for (int d = 0; d < C::DT; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(s_o + (((wave * C::DT + d) * 4 + i) * 64 + lane) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = (o[d][4 * i + e] * f1 + x[e] * f2) * inv;
            // rows 8 i + 4 hf + e of the part
            if (s_nan[out_dim<D>(d, 8 * i + 4 * hf + e)] < lim) y = __uint_as_float(0x7fc00000u);
            o[d][4 * i + e] = y;
          }
        }
      }
      if (rec != nullptr) {
#pragma unroll
        for (int d = 0; d < C::DT; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(rec + (((wave * C::DT + d) * 4 + i) * 64 + lane) * 4) =
                f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        }
        if (hf == 0) {
          rec[kRows * D + (wave * 32 + l32) * 2] = mm;
          rec[kRows * D + (wave * 32 + l32) * 2 + 1] = ll;
        }
      } else if (there) {
        bf16* dst = a.out + (static_cast<size_t>(it.q0 + tok) * a.Hq + h) * D;
        if constexpr (D == 64) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e)   // dims 4 m + {0, 1, 2, 3} from rows m and m + 16 of both parts
              *reinterpret_cast<u32x2*>(dst + 4 * (8 * i + 4 * hf + e)) =
                  u32x2{pack_bf16x2(o[0][4 * i + e], o[0][8 + 4 * i + e]), pack_bf16x2(o[1][4 * i + e], o[1][8 + 4 * i + e])};
          }
        } else {
#pragma unroll
          for (int g = 0; g < D / 128; ++g) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              *reinterpret_cast<u32x2*>(dst + 128 * g + 4 * (8 * (i >> 2) + 4 * hf + (i & 3))) =
                  u32x2{pack_bf16x2(o[4 * g][i], o[4 * g + 1][i]), pack_bf16x2(o[4 * g + 2][i], o[4 * g + 3][i])};
          }
        }
      }
    }
    }
    __syncthreads();   // LDS is the next item's
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
  float M = -INFINITY, L = 0.f;
  for (int x = 0; x < cuts; ++x) M = fmaxf(M, ml[x * step]);
  f32x4 o[4] = {};
  for (int x = 0; x < cuts; ++x) {
    const float m = ml[x * step], f = m == -INFINITY ? 0.f : fast_exp2(m - M);
    L += f * ml[x * step + 1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dt = D == 64 ? e >> 1 : 4 * g + e, quad = D == 64 ? i + 2 * (e & 1) : i;
      o[e] += f * *reinterpret_cast<const f32x4*>(r0 + x * step + (((wave * C::DT + dt) * 4 + quad) * 64 + lane) * 4);
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
// CUs have one, none shorter than kMinRun key tiles where the length is the bound.
void shape(int T, int B, int Hkv, int group, int key_tile, int max_len, int* lanes, int* splits) {
  const int tiles = static_cast<int>((static_cast<long>(T) * group + kRows - 1) / kRows);
  *lanes = std::max(1, kCus / Hkv);
  *splits = 1;
  if (B == 1 && tiles < *lanes) {
    const int runs = std::max(1, (max_len + key_tile - 1) / key_tile / kMinRun);
    *splits = std::min(*lanes / tiles, runs);
  }
}

template <int D>
size_t workspace_need(int T, int B, int Hkv, int group, int max_len, int* lanes, int* splits) {
  shape(T, B, Hkv, group, Cfg<D>::BN, max_len, lanes, splits);
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
    hipLaunchKernelGGL((gqa_prefill_paged_fp8_kernel<D>), dim3(args.lanes * c.Hkv), dim3(kThreads), Cfg<D>::LDS, st, cache, args);
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
    hipLaunchKernelGGL(gqa_prefill_paged_fp8_plan_kernel, dim3(1), dim3(kPlanThreads), static_cast<size_t>(a.B + 1) * sizeof(int), st, a,
                       Cfg<D>::BN);
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
