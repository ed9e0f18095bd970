// Attention of many query rows over the paged 8-bit cache (a prompt's chunk against the context
// before it): the maths of sdpa_kv8.cu on tcgen05 with accumulators in tensor memory.
//
//   t_j = log2(e) scale (q . k_j) 2^ek_j + ev_j,  o = sum_j 2^(t_j - r) v_j / sum_j 2^(t_j - r - ev_j)
//
// Tensor-bound: 4 D operations a row and key, 2 D bytes a key for all rows. One CTA an SM
// covers two 128-row tiles (one at head dim 256, whose output takes half the tensor memory) that
// share every 128-key tile; rows are (token, head of the group), so all heads of a group share
// the keys too. Roles:
//   warps 0-3, 4-7  softmax and epilogue of row tile 0, 1 (thread = row); they also bring the
//                   rows of q into shared memory as fp16 times a power of two (at head dim 256
//                   warps 4-7 are converters of V, and warps 8-11 of K)
//   warps 8-11      converters: codes from the pages straight into registers (up to a tile
//                   ahead), fp16 (exact) into the 128-byte-swizzled tiles that tcgen05 reads, a
//                   unit being one tile's K or V
//   warps 12, 15    MMA issue for row tile 0, 1 (kind::f16, fp16 operands): one thread for both took
//                   longer to issue and wait than the tensor pipe to compute
//   warp 13         walks ahead through line, page table and scales
//   warp 14         zeroes the rows of blocks without keys
// Converting once in shared memory costs 2 D x 128 conversions a tile for 256 rows; fp8
// MMAs would take e4m3 as it is, but then the weights have to be cut into several fp8 parts,
// which costs the softmax warps, the tightest role, about three operations more an element.
// The scales of a page cost nothing an element: softmax's multiply-add takes them 16 keys
// at a time.
//
// Work is a line of key tiles over (sequence, head, block of rows), cut into equal runs, one a
// CTA: causal blocks of different length and uneven sequences fill the GPU evenly. A block that is
// cut leaves partial results, merged by a second kernel that starts before this one ends.
//
// Measured: 2 x 1024 tokens of 32 heads (8 in the cache) at the end of 8192, head dim 128: 319 us,
// 808 TFLOP/s of those that the masks leave. A tile takes some 5000 clocks, of which the MMAs are
// 2 x 634; most stalls are on scores from tensor memory and on fixed latencies, and the walk over the
// line spills (some 580 bytes of loads, with two row tiles). A block's start and end take some
// 18000 (its rows of q, the first scores, the last weights, the output).
//
// Every wait is bounded: on expiry the kernel records TA_DEVSTAT_* bits, drains its MMAs, frees
// tensor memory and returns.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>
#include <utility>

#include "kv8_device.cuh"

namespace ta {
namespace kv8 {
namespace chunk {
namespace {

constexpr int kTileRows = 128, kTileKeys = 128;
constexpr int kHalfKeys = kTileKeys / 2;  // keys of a score half
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kLaunchRegs = 128;
constexpr uint32_t kTmemCols = 512;
constexpr float kBelow = 7.f, kGrowth = 15.f;  // see sdpa_kv8.cu
// t - ref comes out of one multiply-add on the score and so is more exact than ref, which is a rounded t
// less 7: a weight may pass 2^15 by 2^(3 * 2^-24 |ref|), which from |ref| = 2^22 on may pass fp16's 65504.
// A block with a reference beyond kFar goes on in a second form of the loop that rounds t first, as the
// kernel for few rows does. (A branch in the one loop: 2 x 1024 tokens at the end of 8192 374-416 us for 324.)
constexpr float kFar = 1048576.f;
constexpr uint64_t kTimeoutNs = 1000000000ull;  // 1 s per wait
constexpr int kMeta = 8;                       // tiles whose places, pages and scales are kept
constexpr int kGroups = kTileKeys / 16;        // blocks of 16 keys: one page each
constexpr int kSegs = 8;                       // segments that are kept

template <int D>
struct Cfg {
  static constexpr int kTiles = D == 256 ? 1 : 2;
  static constexpr int kRows = kTiles * kTileRows;
  // Register split of the launch's 512 x 128 registers: softmax (a group of 128 threads a row tile),
  // converters (the rest of warps 0-11), the others. With one row tile these have no spills (with two
  // their walk over the line has): 2 x 1024 tokens at the end of 8192, head dim 256, 890 us; with 64 for them 980.
  static constexpr int kSoftmaxRegs = 160, kConvertRegs = 128, kSideRegs = kTiles == 2 ? 64 : 96;
  static_assert(128 * (kTiles * kSoftmaxRegs + (3 - kTiles) * kConvertRegs + kSideRegs) == kThreads * kLaunchRegs,
                "register split must match the launch allocation");
  static constexpr int kTileBytes = kTileRows * D * 2;  // a q tile, or a K or V unit
  static constexpr int kStages = D == 64 ? 6 : D == 128 ? 4 : 2;
  static constexpr int kChunks = D / 16;                // 16-code chunks of a key
  static constexpr int kQOff = 0;
  static constexpr int kKvOff = kTiles * kTileBytes;
  static constexpr int kMetaOff = kKvOff + kStages * kTileBytes;
  static constexpr int kNanOff = kMetaOff + kMeta * kGroups * (16 + 8);
  static constexpr int kBarOff = kNanOff + kSegs * D * 4;
  static constexpr int kBytes = kBarOff + 1024 + 1024;  // slack: 1024-byte alignment
};

struct Meta {   // of 16 keys: their scales in softmax's terms
  float ks;     // scale of K
  float e;      // log2 of V's scale; -inf where there is no key: such keys have no weight
  float back;   // 2^-e
  int unused;
};

// A key tile on the line, as the converters need it; length -1: the run is over.
struct Tile {
  int key0, length, safe, seg;
};

// A block of rows on the line and the part of it that this run has; n = 0: the run is over. Where
// some of its rows do not see a key (keys from `safe` on), that key's value must not reach them
// as 0 * NaN: the converters write such NaNs as zeros and note, for each dim, the first key
// that has one, and the epilogue gives the NaN to the rows that see it.
struct Segment {
  int b, h, rb, t0, n, tiles;  // key tiles [t0, t0 + n) of `tiles`
  int length, count, safe;
  int first_run;               // of those that share the block
};

struct Barriers {
  uint64_t q_full[2], s_full[2][2], p_full[2][2], o_final[2][2];  // [row tile][half]
  uint64_t drain[2];
  uint64_t kv_full[6], kv_empty[6], meta_full[kMeta], meta_empty[kMeta], seg_full[kSegs], seg_empty[kSegs];
  Segment segs[kSegs];
  Tile tiles[kMeta];
  int any_nan[kSegs];
  uint32_t tmem_base;
  int abort_flag;
};
struct Start {  // where the run begins; its memory is the accumulator's notes' (kNanOff) until then
  int64_t scan[kWarps];
  int64_t w;
  int b;
};
static_assert(sizeof(Barriers) <= 1024 && sizeof(Start) <= kSegs * 64 * 4, "shared memory blocks");

// The run's walk over the line, by all lanes of one warp.
template <int D>
struct Walk {
  const AttendParams& p;
  int64_t at, end;  // tiles
  Segment s;
  SeqExtent e;
  __device__ int block() const {
    return block_tiles(e, p.group * p.T, p.group_recip, s.rb * Cfg<D>::kRows, Cfg<D>::kRows, p.causal, kTileKeys);
  }
  __device__ Walk(const AttendParams& pp, int64_t w0, int64_t w1, int b, int64_t before)
      : p(pp), at(w0), end(w1) {
    s.b = b;
    e = extent_of(p, b);
    const int lane = threadIdx.x & 31;
    auto tiles_at = [&](int rb) {
      s.rb = rb;
      return rb < p.row_blocks ? block() : 0;
    };
    int64_t head = 0;  // tiles of one head
    for (int base = 0; base < p.row_blocks; base += 32)
      head += __reduce_add_sync(0xffffffffu, tiles_at(base + lane));
    int64_t rem = w0 - before;
    s.h = static_cast<int>(rem / head);
    rem -= s.h * head;
    for (int base = 0;; base += 32) {
      const int mine = tiles_at(base + lane);
      int incl = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, incl > rem);
      if (past) {
        const int at_lane = __ffs(past) - 1;
        s.tiles = __shfl_sync(0xffffffffu, mine, at_lane);
        rem -= __shfl_sync(0xffffffffu, incl, at_lane) - s.tiles;
        s.rb = base + at_lane;
        break;
      }
      rem -= __shfl_sync(0xffffffffu, incl, 31);
    }
    begin(static_cast<int>(rem));
  }
  __device__ void begin(int t0) {
    s.t0 = t0;
    s.n = static_cast<int>(min(end - at, static_cast<int64_t>(s.tiles - t0)));
    s.length = e.length;
    s.count = e.count;
    s.safe = e.length;
    if (p.causal) {  // the first token with any keys sees the fewest
      const int tok = max(group_of(p, s.rb * Cfg<D>::kRows), e.count - e.length);
      s.safe = row_limit(e.length, e.count, tok, 1);
    }
  }
  __device__ bool next() {
    at += s.n;
    if (at >= end) return false;
    do {  // the next block with any tiles; there is one, since the run goes on
      if (++s.rb == p.row_blocks) {
        s.rb = 0;
        if (++s.h == p.Hkv) {
          s.h = 0;
          if (++s.b >= p.B) return false;
          e = extent_of(p, s.b);
        }
      }
      s.tiles = block();
    } while (s.tiles == 0);
    begin(0);
    return true;
  }
};

// Whether the second row tile of a block has any rows.
template <int D>
__device__ __forceinline__ bool has_two(const AttendParams& p, int rb) {
  return Cfg<D>::kTiles == 2 && p.group * p.T - rb * Cfg<D>::kRows > kTileRows;
}

__device__ __forceinline__ bool is_far(float ref) { return fabsf(ref) > kFar && ref != -INFINITY; }

__device__ __forceinline__ void report(const AttendParams& p, uint32_t code, volatile int* abort_flag) {
  *abort_flag = 1;
  if (p.status) atomicOr(p.status, code);
}

// The MMAs of a product, descriptor steps as immediates: scores over D dims, 16 at a time (64 dims
// are one 128-byte-wide part of a tile) ...
template <int... kk>
__device__ __forceinline__ void issue_qk_seq(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             std::integer_sequence<int, kk...>) {
  (mma_ss_imm<(((kk >> 2) * (kTileRows * 128) + (kk & 3) * 32) >> 4),
              (((kk >> 2) * (kTileKeys * 128) + (kk & 3) * 32) >> 4), (kk > 0 ? 1 : 0)>(d, a, b, idesc),
   ...);
}
// ... and the output over keys, 16 at a time.
template <int... kk>
__device__ __forceinline__ void issue_pv_seq(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                             uint32_t acc, std::integer_sequence<int, kk...>) {
  (mma_ts_imm_acc<kk * 8, ((kk * 16 * 128) >> 4)>(d, a, b, idesc, kk == 0 ? acc : 1u), ...);
}

__device__ __forceinline__ void st_shared128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w));
}

__device__ __forceinline__ void sts128(void* a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  *reinterpret_cast<uint4*>(a) = make_uint4(x, y, z, w);
}

__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const AttendParams p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* q_smem = smem + C::kQOff;
  uint8_t* kv_smem = smem + C::kKvOff;
  Meta* meta = reinterpret_cast<Meta*>(smem + C::kMetaOff);
  // Where 16 keys are: byte offset of the first one's codes * 32 + how many there are.
  int64_t* place = reinterpret_cast<int64_t*>(meta + kMeta * kGroups);
  int* nan_key = reinterpret_cast<int*>(smem + C::kNanOff);  // [kSegs][D]
  Start* start = reinterpret_cast<Start*>(nan_key);
  Barriers* bars = reinterpret_cast<Barriers*>(smem + C::kBarOff);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_stream();

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], kTileRows);
      for (int half = 0; half < 2; ++half) {
        mbar_init(&bars->s_full[t][half], 1);
        mbar_init(&bars->p_full[t][half], kTileRows);
        mbar_init(&bars->o_final[t][half], 1);
      }
    }
    mbar_init(&bars->drain[0], 1);
    mbar_init(&bars->drain[1], 1);
    start->b = -1;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->kv_full[s], 128);
      mbar_init(&bars->kv_empty[s], C::kTiles);
    }
    for (int i = 0; i < kMeta; ++i) {
      mbar_init(&bars->meta_full[i], 32);
      mbar_init(&bars->meta_empty[i], C::kTiles);
    }
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&bars->seg_full[i], 32);
      mbar_init(&bars->seg_empty[i], 5 * C::kTiles);  // a row tile's softmax and MMA warps
    }
    bars->abort_flag = 0;
    p.cuts[blockIdx.x] = Cut{0, 0, 0, -1};  // until this thread knows better
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  // Items: blocks of rows of one head of each sequence.
  const auto item_work = [&](int i) {
    const int b = i / p.row_blocks, rb = i - b * p.row_blocks;
    const SeqExtent e = extent_of(p, b);
    if (rb == 0) report_extent(p, e);
    return static_cast<int64_t>(block_tiles(e, p.group * p.T, p.group_recip, rb * C::kRows, C::kRows,
                                            p.causal, kTileKeys)) * p.Hkv;
  };
  const Scan sc = scan_items<kWarps>(p.B * p.row_blocks, start->scan, item_work);  // has a barrier
  tc_fence_after();
  let_next_kernel_in();
  const uint32_t tmem = bars->tmem_base;
  const int64_t parts = min(static_cast<int64_t>(gridDim.x), sc.total);
  const bool has_run = blockIdx.x < parts;
  const int64_t w0 = has_run ? run_begin(blockIdx.x, sc.total, parts) : 0;
  const int64_t w1 = has_run ? run_begin(blockIdx.x + 1, sc.total, parts) : 0;
  // The run's first sequence: the last one whose work begins at or before it.
  if (has_run)
    for (int pass = 0; pass < 2; ++pass) {
      int64_t at = sc.mine;
      for (int i = sc.i0; i < sc.i1; ++i) {
        if (i % p.row_blocks == 0 && at <= w0) {
          if (pass == 0) atomicMax(&start->b, i / p.row_blocks);
          else if (start->b == i / p.row_blocks) start->w = at;
        }
        if (at > w0) break;
        if (pass == 0 || i + 1 < sc.i1) at += item_work(i);
      }
      __syncthreads();
    }

  if (warp >= 12) {
    regs_dec<C::kSideRegs>();
    if (warp == 12 || (warp == 15 && C::kTiles == 2)) {
      // ------------------------------------------------------------ MMA issuers
      if (lane == 0 && has_run) {
        constexpr uint32_t kIdescQK = idesc_f16(kTileRows, kHalfKeys, false, false, false);
        constexpr uint32_t kIdescPV = idesc_f16(kTileRows, D, false, false, true);
        constexpr uint32_t kUnit = C::kTileBytes >> 4;  // in a descriptor's 16-byte steps
        constexpr uint32_t kHalfStep = kHalfKeys * 128 >> 4;
        const int t = warp == 12 ? 0 : 1;
        const uint64_t q_desc = sdesc_sw128(smem_u32(q_smem + t * C::kTileBytes), 16, 1024);
        const uint64_t kv_desc_k = sdesc_sw128(smem_u32(kv_smem), 16, 1024);
        const uint64_t kv_desc_v = sdesc_sw128(smem_u32(kv_smem), kTileKeys * 128, 1024);
        const uint32_t t_s = tmem + t * 128, t_o = tmem + 256 + t * D;
        uint64_t* const s_full = bars->s_full[t];
        uint64_t* const p_full = bars->p_full[t];
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          if (!mbar_try_wait(smem_u32(bar), parity))
            ok = ok && mbar_wait_bounded(bar, parity, abort_flag, kTimeoutNs);
          tc_fence_after();
          return ok;
        };
        uint32_t st = 0, phase = 0;  // of the next unit
        auto next_unit = [&]() {
          if (++st == C::kStages) {
            st = 0;
            phase ^= 1;
          }
        };
        // Halves: a row tile's columns of tensor memory hold the scores of two times 64 keys, so the
        // next tile's first half is computed while softmax works on this one's second.
        auto issue_qk = [&](int half, uint64_t kd) {
          issue_qk_seq(t_s + half * kHalfKeys, q_desc, kd + half * kHalfStep, kIdescQK,
                       std::make_integer_sequence<int, D / 16>());
          mma_commit(&s_full[half]);
        };
        uint32_t q_par = 0, p_par = 0;
        int tile_no = 0;
        for (int seg = 0; ok; ++seg) {
          if (!wait(&bars->seg_full[seg % kSegs], (seg / kSegs) & 1)) break;
          const int n = bars->segs[seg % kSegs].n;
          const bool mine = t == 0 || has_two<D>(p, bars->segs[seg % kSegs].rb);
          mbar_arrive(&bars->seg_empty[seg % kSegs]);
          if (n == 0) break;
          if (!mine) {  // no rows: the units pass
            for (int u = 0; ok && u < 2 * n; ++u) {
              if (!wait(&bars->kv_full[st], phase)) break;
              mbar_arrive(&bars->kv_empty[st]);
              next_unit();
              if (u & 1) mbar_arrive(&bars->meta_empty[tile_no++ % kMeta]);
            }
            continue;
          }
          wait(&bars->q_full[t], q_par);
          q_par ^= 1;
          if (!wait(&bars->kv_full[st], phase)) break;
          issue_qk(0, kv_desc_k + st * kUnit);
          issue_qk(1, kv_desc_k + st * kUnit);
          mma_commit(&bars->kv_empty[st]);
          next_unit();
          for (int j = 0; j < n; ++j) {
            const uint32_t st_v = st;
            const uint64_t vd = kv_desc_v + st * kUnit;
            wait(&bars->kv_full[st], phase);
            next_unit();
            const bool more = j + 1 < n;
            const uint64_t kd = kv_desc_k + st * kUnit;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (!wait(&p_full[half], p_par)) break;
              issue_pv_seq(t_o, t_s + half * kHalfKeys, vd + half * kHalfStep, kIdescPV,
                           half > 0 || j > 0 ? 1u : 0u, std::make_integer_sequence<int, kHalfKeys / 16>());
              if (more) {
                if (half == 0 && !wait(&bars->kv_full[st], phase)) break;
                issue_qk(half, kd);
              } else {
                mma_commit(&bars->o_final[t][half]);
              }
            }
            if (!ok) break;
            mma_commit(&bars->kv_empty[st_v]);
            if (more) {
              mma_commit(&bars->kv_empty[st]);
              next_unit();
            }
            p_par ^= 1;
            // Softmax has taken this tile's scales and the converters its pages.
            mbar_arrive(&bars->meta_empty[tile_no++ % kMeta]);
          }
        }
        if (!ok && !*abort_flag) report(p, TA_DEVSTAT_TIMEOUT_MMA, abort_flag);
        // All MMAs this thread issued complete before tensor memory is freed.
        mma_commit(&bars->drain[t]);
        volatile int no_abort = 0;
        if (!mbar_wait_bounded(&bars->drain[t], 0, &no_abort, kTimeoutNs) && p.status)
          atomicOr(p.status, TA_DEVSTAT_TIMEOUT_DRAIN);
      }
      __syncwarp();
    } else if (warp == 13) {
      // ------------------------------------------------------------ pages and scales
      // Lane i < 8: block i of 16 keys of a tile. Page ids are fetched two tiles and scales one
      // tile before they are published.
      if (has_run) {
        const int64_t before = start->w;
        Walk<D> w(p, w0, w1, start->b, before);
        __syncwarp();  // `start` may be written over
        bool ok = true;
        int seg = 0, j = 0;
        auto wait = [&](uint64_t* bar, int parity) {
          ok = mbar_wait_bounded(bar, parity & 1, abort_flag, kTimeoutNs);
          ok = __all_sync(0xffffffffu, ok);
          return ok;
        };
        auto publish_segment = [&](bool over) {
          const int slot = seg % kSegs;
          if (!wait(&bars->seg_empty[slot], (seg / kSegs) ^ 1)) return;
          if (lane == 0) {
            Segment& to = bars->segs[slot];
            to = w.s;
            if (over) to.n = 0;
            else to.first_run = static_cast<int>(run_of(w.at - w.s.t0, sc.total, parts));
            bars->any_nan[slot] = 0;
          }
          for (int d = lane; d < D; d += 32) nan_key[slot * D + d] = 0x7fffffff;
          mbar_arrive(&bars->seg_full[slot]);
          ++seg;
        };
        struct Ahead {
          int id;       // page id, -1: no key, -2: outside the cache
          int h;
          Tile tile;    // length -1: none
        };
        bool more = true;
        auto next_tile = [&]() {  // of the run, and on; its segment is published first
          Ahead a{-1, 0, {0, -1, 0, 0}};
          if (!more) return a;
          if (j == 0) publish_segment(false);
          if (!ok) return a;
          a.h = w.s.h;
          a.tile = Tile{(w.s.t0 + j) * kTileKeys, w.s.length, w.s.safe, seg - 1};
          const uint32_t key = static_cast<uint32_t>(a.tile.key0) + lane * 16;
          if (lane < kGroups && key < static_cast<uint32_t>(w.s.length)) {
            a.id = p.table[w.s.b * p.table_stride + (key >> p.page_shift)];
            if (static_cast<unsigned>(a.id) >= static_cast<unsigned>(p.num_pages)) a.id = -2;
          }
          if (++j == w.s.n) {
            j = 0;
            more = w.next();
          }
          return a;
        };
        float ks = 1.f, vs = 1.f;
        auto fetch_scales = [&](const Ahead& a) {
          if (a.id >= 0) {
            const int64_t plane = static_cast<int64_t>(a.id) * p.Hkv + a.h;
            ks = p.scale[0][plane];
            vs = p.scale[1][plane];
          }
        };
        Ahead a0 = next_tile();
        Ahead a1 = next_tile();
        fetch_scales(a0);
        for (int n = 0; ok; ++n) {
          Meta m{1.f, -INFINITY, 0.f, 0};
          int64_t at = 0;
          if (a0.id >= 0) {
            const ValueScale v = value_scale(__float_as_uint(vs));
            m = Meta{ks, v.e, v.back, 0};
            const int key = a0.tile.key0 + lane * 16;
            const int64_t row = (static_cast<int64_t>(a0.id) * p.Hkv + a0.h) * p.page + (key & (p.page - 1));
            at = row * p.D * 32 + min(16, a0.tile.length - key);
          } else if (a0.id == -2 && p.status) {
            atomicOr(p.status, TA_DEVSTAT_BAD_PAGE);
          }
          const Tile now = a0.tile;
          a0 = a1;
          if (ok && now.length >= 0) a1 = next_tile();
          fetch_scales(a0);
          if (!ok || !wait(&bars->meta_empty[n % kMeta], (n / kMeta) ^ 1)) break;
          if (lane < kGroups) {
            meta[(n % kMeta) * kGroups + lane] = m;
            place[(n % kMeta) * kGroups + lane] = at;
          }
          if (lane == 0) bars->tiles[n % kMeta] = now;
          mbar_arrive(&bars->meta_full[n % kMeta]);
          if (now.length < 0) break;
        }
        if (ok) publish_segment(true);
        if (!ok && lane == 0 && !*abort_flag) report(p, TA_DEVSTAT_TIMEOUT_LOAD, abort_flag);
      }
    } else if (warp == 14) {
      // ------------------------------------------------------------ rows of blocks without keys
      const int rows = p.group * p.T;
      const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * p.row_blocks;
      for (int64_t i = blockIdx.x; i < blocks; i += gridDim.x) {
        const int rb = static_cast<int>(i % p.row_blocks);
        const int h = static_cast<int>(i / p.row_blocks % p.Hkv);
        const int b = static_cast<int>(i / p.row_blocks / p.Hkv);
        if (block_tiles(extent_of(p, b), rows, p.group_recip, rb * C::kRows, C::kRows, p.causal, kTileKeys))
          continue;
        const int r1 = min(rows, (rb + 1) * C::kRows);
        for (int r = rb * C::kRows; r < r1; ++r) {
          const int tok = group_of(p, r), hd = h * p.group + (r - tok * p.group);
          uint16_t* out = static_cast<uint16_t*>(p.o) + b * p.o_sb + hd * p.o_sh + tok * p.o_ss;
          for (int d = lane * 8; d < p.D; d += 256) sts128(out + d, 0, 0, 0, 0);
          if (p.lse && lane == 0)
            p.lse[(static_cast<int64_t>(b) * p.Hq + hd) * p.T + tok] = -INFINITY;
        }
      }
    }
  } else if (warp >= (C::kTiles == 2 ? 8 : 4)) {
    // ------------------------------------------------------------ converters
    regs_dec<C::kConvertRegs>();
    if (has_run) {
      constexpr int kRowsPerPass = 128 / C::kChunks;  // of 128 threads, 16 codes each
      // The passes of a tile are in flight, of K and V, or where the second row tile's warps convert too
      // of one of them: those warps V, the others K. (Warps 8-11 alone, a unit in flight: 2 x 1024
      // tokens at the end of 8192, 32 heads over 8, head dim 256: 1102 us, so 921.)
      constexpr int kKinds = C::kTiles == 2 ? 2 : 1;
      static_assert(kKinds == 2 || C::kStages == 2, "a stage for K and one for V");
      const int first_kind = warp < 8 ? 1 : 0;
      constexpr int kHeld = kKinds * C::kChunks;
      // Lanes: 4 chunks of one 128-byte row of the tile and the next key's, so that 8
      // lanes' 16-byte stores meet 8 different banks.
      const int c = (lane & 3) | (C::kChunks == 4 ? 0 : (lane >> 3 & (C::kChunks / 4 - 1)) << 2);
      const int row_in_warp = C::kChunks == 4 ? lane >> 2
                              : C::kChunks == 8 ? ((lane >> 2) & 1) | (lane >> 4 << 1)
                                                : (lane >> 2) & 1;
      const int row0 = (warp & 3) * (kRowsPerPass / 4) + row_in_warp;
      const bool real = c * 16 < p.D;
      const uint32_t store = smem_u32(kv_smem) + (c >> 2) * (kTileKeys * 128);  // 64 dims: 128 bytes a key
      // The thread's two 16-byte pieces of a row, swizzled; a pass's rows are 8 k apart or more.
      const uint32_t piece0 = row0 * 128 + ((((2 * c) & 7) ^ (row0 & 7)) << 4);
      const uint32_t piece1 = row0 * 128 + ((((2 * c + 1) & 7) ^ (row0 & 7)) << 4);
      static_assert(kRowsPerPass % 8 == 0, "a pass keeps a row's swizzle");
      constexpr int kPlaces = kRowsPerPass >= 16 ? C::kChunks : C::kChunks / 2;
      const uint32_t places = smem_u32(place) + (kRowsPerPass > 16 ? row0 >> 4 : 0) * 8;
      const int in_block = row0 & 15;
      const uint8_t* const mine[2] = {p.pages[first_kind] + in_block * p.D + c * 16,
                                      p.pages[1] + in_block * p.D + c * 16};
      bool ok = true;
      int st = first_kind, phase = 0;  // of the next unit

      int64_t at[kPlaces];  // of the tile whose codes are loaded next
      auto read_places = [&](int slot) {
#pragma unroll
        for (int i = 0; i < kPlaces; ++i)
          asm volatile("ld.shared.b64 %0, [%1];"
                       : "=l"(at[i])
                       : "r"(places + (slot * kGroups + i * (kRowsPerPass > 16 ? kRowsPerPass / 16 : 1)) * 8));
      };
      // Codes of pass i of the u-th unit here of that tile. Rows without a key read as zeros.
      auto fetch = [&](int i, int u) {
        const int64_t where = at[kRowsPerPass >= 16 ? i : i / 2];
        const int row = in_block + (kRowsPerPass < 16 ? (i & 1) * kRowsPerPass : 0);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (real && row < static_cast<int>(where & 31))
          v = __ldg(reinterpret_cast<const uint4*>(mine[u] + (where >> 5) + (row - in_block) * p.D));
        return v;
      };
      auto wait_meta = [&](int n) {
        return mbar_wait_bounded(&bars->meta_full[n % kMeta], (n / kMeta) & 1, abort_flag, kTimeoutNs);
      };

      uint4 held[kHeld];
      ok = wait_meta(0);
      Tile now{0, -1, 0, 0};
      if (ok) {
        now = bars->tiles[0];
        read_places(0);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = fetch(i % C::kChunks, i / C::kChunks);
      }
      for (int tile_no = 1; ok && now.length >= 0; ++tile_no) {
        const int key0 = now.key0;
        const bool edge = key0 > now.safe - kTileKeys;  // values that some row does not see
        int* const nan_here = nan_key + now.seg % kSegs * D;
        int* const any_nan = &bars->any_nan[now.seg % kSegs];
        ok = wait_meta(tile_no);  // the next tile's pages
        if (!ok) break;
        now = bars->tiles[tile_no % kMeta];
        read_places(tile_no % kMeta);
#pragma unroll
        for (int u = 0; u < kKinds; ++u) {
          const int kind = kKinds == 2 ? u : first_kind;  // 0 K, 1 V
          ok = ok && mbar_wait_bounded(&bars->kv_empty[st], phase ^ 1, abort_flag, kTimeoutNs);
          if (!ok) break;
          const uint32_t dst = store + st * C::kTileBytes;
          uint32_t nans = 0;
#pragma unroll
          for (int i = 0; i < C::kChunks; ++i) {
            const uint4 v = held[u * C::kChunks + i];
            if (kind == 1) nans |= nan_bits(v.x) | nan_bits(v.y) | nan_bits(v.z) | nan_bits(v.w);
            uint32_t f[8];
            codes_to_f16(v.x, f[0], f[1]);
            codes_to_f16(v.y, f[2], f[3]);
            codes_to_f16(v.z, f[4], f[5]);
            codes_to_f16(v.w, f[6], f[7]);
            st_shared128(dst + i * (kRowsPerPass * 128) + piece0, f[0], f[1], f[2], f[3]);
            st_shared128(dst + i * (kRowsPerPass * 128) + piece1, f[4], f[5], f[6], f[7]);
          }
          if (kind == 1 && edge && nans) {  // rare: over the thread's own values once more
#pragma unroll 1
            for (int i = 0; i < C::kChunks * 16; ++i) {
              const int pass = i >> 4, k = i & 15;
              const uint32_t a = dst + pass * (kRowsPerPass * 128) + (k < 8 ? piece0 : piece1) + (k & 7) * 2;
              uint16_t h;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(a));
              if ((h & 0x7fff) <= 0x7c00) continue;
              *any_nan = 1;
              atomicMin(nan_here + c * 16 + k, key0 + pass * kRowsPerPass + row0);
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(static_cast<uint16_t>(0)));
            }
          }
          fence_proxy_async_shared();
          mbar_arrive(&bars->kv_full[st]);
          // The registers' next loads, the next tile's. All in one burst: a load issued between the uses
          // of others makes those uses wait for it too.
#pragma unroll
          for (int i = 0; i < C::kChunks; ++i) held[u * C::kChunks + i] = fetch(i, u);
          if (kKinds == 1) {
            phase ^= 1;
          } else if (++st == C::kStages) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && threadIdx.x % 128 == 0 && !*abort_flag) report(p, TA_DEVSTAT_TIMEOUT_LOAD, abort_flag);
    }
  } else {
    regs_inc<C::kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax + epilogue
    const int t = warp >> 2;  // row tile of this warpgroup
    if (t < C::kTiles && has_run) {
      const int quarter = warp & 3;  // TMEM lanes this warp may access
      const int r_in_tile = quarter * 32 + lane;
      const uint32_t lane_bits = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t t_s = tmem + lane_bits + t * 128;
      const uint32_t t_o = tmem + lane_bits + 256 + t * D;
      const int rows = p.group * p.T;
      bool ok = true;
      int tile_no = 0, seen = 0, segs = 0;  // tiles of the run, halves and blocks of this row tile
      for (int seg = 0; ok; ++seg) {
        const int seg_slot = seg % kSegs;
        ok = mbar_wait_bounded(&bars->seg_full[seg_slot], (seg / kSegs) & 1, abort_flag, kTimeoutNs);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0 && !*abort_flag) report(p, TA_DEVSTAT_TIMEOUT_SOFTMAX, abort_flag);
          break;
        }
        const Segment s = bars->segs[seg_slot];
        if (s.n == 0) break;
        if (t == 1 && !has_two<D>(p, s.rb)) {
          tile_no += s.n;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->seg_empty[seg_slot]);
          continue;
        }
        const int row = s.rb * C::kRows + t * kTileRows + r_in_tile;
        const int tok = group_of(p, row), hd = s.h * p.group + (row - tok * p.group);
        const bool real = row < rows && tok < s.count;
        const int lim = real ? row_limit(s.length, s.count, tok, p.causal) : 0;
        const int safe = __reduce_min_sync(0xffffffffu, lim > 0 ? lim : 0x7fffffff);

        // The row of q times a power of two, with its largest value in [2^14, 2^15), as fp16.
        float mul;
        {
          const uint4* q = reinterpret_cast<const uint4*>(
              static_cast<const uint16_t*>(p.q) + s.b * p.q_sb + static_cast<int64_t>(hd) * p.q_sh +
              static_cast<int64_t>(tok) * p.q_ss);
          constexpr int kOnce = D <= 128 ? D / 8 : 16;  // vectors held at a time
          uint4 v[kOnce];
          float amax = 0.f;
          auto load = [&](int base) {
#pragma unroll
            for (int i = 0; i < kOnce; ++i) {
              v[i] = make_uint4(0, 0, 0, 0);
              if (real && (base + i) * 8 < p.D) v[i] = q[base + i];
            }
          };
#pragma unroll 1
          for (int base = 0; base < D / 8; base += kOnce) {
            load(base);
#pragma unroll
            for (int i = 0; i < kOnce; ++i) {
              const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 a = unpack16(x[k], p.bf16);
                amax = fmaxf(amax, fmaxf(fabsf(a.x), fabsf(a.y)));
              }
            }
          }
          const int ex = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 14, -126), 113);
          const float up = row_factor(amax, ex);
          mul = p.scale_log2 * pow2f(ex);
          uint8_t* dst = q_smem + t * C::kTileBytes + r_in_tile * 128;
#pragma unroll 1
          for (int base = 0; base < D / 8; base += kOnce) {
            if (D / 8 > kOnce) load(base);
#pragma unroll
            for (int i = 0; i < kOnce; ++i) {
              const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
              uint32_t y[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 a = unpack16(x[k], p.bf16);
                y[k] = pack_f16(a.x * up, a.y * up);
              }
              sts128(dst + ((base + i) >> 3) * (kTileRows * 128) + ((i & 7) ^ (r_in_tile & 7)) * 16, y[0],
                     y[1], y[2], y[3]);
            }
          }
          fence_proxy_async_shared();
          mbar_arrive(&bars->q_full[t]);
        }

        float ref = -INFINITY, l_run = 0.f;
        // The block's halves from j2 on; the first that was not finished.
        auto halves = [&](auto far_rows, int j2) {
          constexpr bool kFarRows = decltype(far_rows)::value;
          for (; j2 < 2 * s.n; ++j2, ++seen) {
            const int half = j2 & 1;
            const int slot = tile_no % kMeta;
            if (half == 0)
              ok = mbar_wait_bounded(&bars->meta_full[slot], (tile_no / kMeta) & 1, abort_flag, kTimeoutNs);
            ok = ok && mbar_wait_bounded(&bars->s_full[t][half], (seen >> 1) & 1, abort_flag, kTimeoutNs);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return j2;
            tc_fence_after();
            uint32_t x[64];
            tmem_ld64(t_s + half * kHalfKeys, *reinterpret_cast<uint32_t(*)[32]>(x),
                      *reinterpret_cast<uint32_t(*)[32]>(x + 32));
            tmem_wait_ld();
            const int key0 = (s.t0 + (j2 >> 1)) * kTileKeys + half * kHalfKeys;
            if (key0 > safe - kHalfKeys) {
              const int visible = lim - key0;
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (i >= visible) x[i] = 0xff800000u;
            }
            const Meta* m = meta + slot * kGroups + half * (kGroups / 2);
            // t = score * c + e, c held above zero so that a masked score stays -inf
            float cand = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float a = fmaxf(__uint_as_float(x[16 * g]), __uint_as_float(x[16 * g + 1]));
              float b = fmaxf(__uint_as_float(x[16 * g + 2]), __uint_as_float(x[16 * g + 3]));
#pragma unroll
              for (int i = 4; i < 16; i += 4) {
                a = fmax3(a, __uint_as_float(x[16 * g + i]), __uint_as_float(x[16 * g + i + 1]));
                b = fmax3(b, __uint_as_float(x[16 * g + i + 2]), __uint_as_float(x[16 * g + i + 3]));
              }
              cand = fmaxf(cand, fmaf(fmaxf(a, b), fmaxf(mul * m[g].ks, 1e-37f), m[g].e));
            }
            const bool grow = cand - ref > kGrowth;  // not cand > ref + kGrowth, a sum that may round up
            if (__any_sync(0xffffffffu, grow)) {
              float alpha = 1.f;
              if (grow) {
                alpha = ex2_approx(ref - (cand - kBelow));  // 0 from -inf
                ref = cand - kBelow;
                l_run *= alpha;
              }
              if (j2 > 0) {
                // The product of the half before may still be adding to the output. Behind it come the
                // scores of the half after this one, or in the last tile its own signal.
                ok = j2 + 1 < 2 * s.n
                         ? mbar_wait_bounded(&bars->s_full[t][half ^ 1], ((seen + 1) >> 1) & 1, abort_flag, kTimeoutNs)
                         : mbar_wait_bounded(&bars->o_final[t][0], segs & 1, abort_flag, kTimeoutNs);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return j2;
                tc_fence_after();
                const uint64_t alpha2 = f2_pack(alpha, alpha);
#pragma unroll 1
                for (int cc = 0; cc < D / 32; ++cc) {
                  uint32_t o[32];
                  tmem_ld32(t_o + cc * 32, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 32; i += 2) {
                    float a0, a1;
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), alpha2),
                              a0, a1);
                    o[i] = __float_as_uint(a0);
                    o[i + 1] = __float_as_uint(a1);
                  }
                  tmem_st32(t_o + cc * 32, o);
                }
              }
              if (!kFarRows && __any_sync(0xffffffffu, is_far(ref))) return j2;  // this half in the other form
            }
            if (kFarRows && is_far(ref)) {  // t - ref in the scores' place, as what gives it without ref
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const float cs = fmaxf(mul * m[g].ks, 1e-37f), inv = 1.f / cs;
                const float e = m[g].e, finite_e = fmaxf(e, -1e3f);
#pragma unroll
                for (int i = 16 * g; i < 16 * g + 16; ++i)
                  x[i] = __float_as_uint((fmaf(__uint_as_float(x[i]), cs, e) - ref - finite_e) * inv);
              }
            }
            // The weights (16-bit, two a column) go over the first 32 of the half's columns.
            const float r = ref == -INFINITY || (kFarRows && is_far(ref)) ? 0.f : ref;
            uint32_t pk[32];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float cs = fmaxf(mul * m[g].ks, 1e-37f), sh = m[g].e - r;
              const uint64_t c2 = f2_pack(cs, cs), s2 = f2_pack(sh, sh);
              uint64_t sum = f2_pack(0.f, 0.f);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float a0, a1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(x[16 * g + 2 * i]),
                                         __uint_as_float(x[16 * g + 2 * i + 1])), c2, s2), a0, a1);
                a0 = ex2_approx(a0);
                a1 = ex2_approx(a1);
                pk[g * 8 + i] = pack_f16(a0, a1);
                sum = f2_add(sum, f2_pack(a0, a1));
              }
              float s0, s1;
              f2_unpack(sum, s0, s1);
              l_run = fmaf(s0 + s1, m[g].back, l_run);
            }
            tmem_st32(t_s + half * kHalfKeys, pk);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars->p_full[t][half]);
            tile_no += half;
          }
          return j2;
        };
        const int far_from = halves(std::false_type(), 0);
        if (ok && far_from < 2 * s.n) halves(std::true_type(), far_from);
        if (ok) {  // the last tile's products
          ok = mbar_wait_bounded(&bars->o_final[t][0], segs & 1, abort_flag, kTimeoutNs) &&
               mbar_wait_bounded(&bars->o_final[t][1], segs & 1, abort_flag, kTimeoutNs);
          ++segs;
          ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok) {
          if (lane == 0 && !*abort_flag) report(p, TA_DEVSTAT_TIMEOUT_SOFTMAX, abort_flag);
          break;
        }
        tc_fence_after();
        const bool whole = s.n == s.tiles;
        if (lim == 0) {  // a row without keys: its unmasked scores were of no row
          ref = -INFINITY;
          l_run = 0.f;
        }
        const bool has = ref != -INFINITY;
        const float inv = !whole ? 1.f : l_run == 0.f ? 0.f : 1.f / l_run;
        // Partial results: [run][first or last block][4 dims][row][4], so that a warp's rows are
        // written and read side by side.
        const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (s.t0 == 0 ? 1 : 0)) * C::kRows;
        uint16_t* out = static_cast<uint16_t*>(p.o) + s.b * p.o_sb + static_cast<int64_t>(hd) * p.o_sh +
                        static_cast<int64_t>(tok) * p.o_ss;
        const bool any_nan = *static_cast<volatile int*>(&bars->any_nan[seg_slot]) != 0;
        const int* nan_here = nan_key + seg_slot * D;
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t o[32];
          tmem_ld32(t_o + cc * 32, o);
          tmem_wait_ld();
          if (any_nan) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (nan_here[cc * 32 + i] < lim) o[i] = 0x7fffffffu;
          }
          if (row < rows) {
            if (!whole) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                if (cc * 32 + i < p.D)
                  *reinterpret_cast<float4*>(p.part_o + part * D +
                                             ((cc * 8 + i / 4) * C::kRows + t * kTileRows + r_in_tile) * 4) =
                      has ? make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]),
                                        __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 8)
                if (cc * 32 + i < p.D) {
                  uint32_t y[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const float a = has ? __uint_as_float(o[i + 2 * k]) : 0.f;
                    const float b = has ? __uint_as_float(o[i + 2 * k + 1]) : 0.f;
                    y[k] = pack16(a * inv, b * inv, p.bf16);
                  }
                  sts128(out + cc * 32 + i, y[0], y[1], y[2], y[3]);
                }
            }
          }
        }
        if (row < rows) {
          if (!whole)
            *reinterpret_cast<float2*>(p.part_ml + (part + t * kTileRows + r_in_tile) * 2) =
                make_float2(ref, l_run);
          else if (p.lse)
            p.lse[(static_cast<int64_t>(s.b) * p.Hq + hd) * p.T + tok] = lse_of(ref, l_run);
        }
        // The run that ends a cut block leaves its merge's address.
        if (t == 0 && threadIdx.x == 0 && s.t0 > 0 && s.t0 + s.n == s.tiles) {
          p.cuts[blockIdx.x] = Cut{s.b, s.h, s.rb, s.first_run};
        }
        // The next block's MMAs write the accumulator that was just read.
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->seg_empty[seg_slot]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, kTmemCols);
}

// Merges the blocks that several runs share: blockIdx.x = the run that ends the block,
// blockIdx.y = 32 of its rows, a lane each; a warp has every eighth group of 4 dims.
template <int D>
__global__ void __launch_bounds__(256) merge_kernel(const AttendParams p) {
  using C = Cfg<D>;
  constexpr int kVec = D / 32;
  constexpr int kStride = D + 8;  // of a row of the 16-bit tile, values
  __shared__ __align__(16) uint16_t tile[32 * kStride];
  wait_for_stream();
  const Cut cut = p.cuts[blockIdx.x];
  if (cut.first < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = min(p.group * p.T - cut.rb * C::kRows, C::kRows);
  const int r0 = blockIdx.y * 32;
  if (r0 >= rows) return;
  const int r = min(r0 + lane, rows - 1);
  float m = -INFINITY, l = 0.f;
  float4 a[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int i = cut.first; i <= static_cast<int>(blockIdx.x); ++i) {
    // the block's first run has it in its second slot, the others in their first
    const int64_t part = (static_cast<int64_t>(i) * 2 + (i == cut.first ? 1 : 0)) * C::kRows;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (part + r) * 2);
    // without a reference: sums of 0 or NaN and outputs of 0, kept as they are
    const float mn = fmaxf(m, ml.x);
    const float fa = m == -INFINITY ? 1.f : exp2f(m - mn);
    const float fb = ml.x == -INFINITY ? 1.f : exp2f(ml.x - mn);
    l = l * fa + ml.y * fb;
    m = mn;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int d4 = v * 8 + warp;
      if (d4 * 4 < p.D) {
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + part * D + (d4 * C::kRows + r) * 4);
        a[v].x = a[v].x * fa + x.x * fb;
        a[v].y = a[v].y * fa + x.y * fb;
        a[v].z = a[v].z * fa + x.z * fb;
        a[v].w = a[v].w * fa + x.w * fb;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int v = 0; v < kVec; ++v)
    *reinterpret_cast<uint2*>(tile + lane * kStride + (v * 8 + warp) * 4) =
        make_uint2(pack16(a[v].x * inv, a[v].y * inv, p.bf16), pack16(a[v].z * inv, a[v].w * inv, p.bf16));
  const int n = min(32, rows - r0);
  auto place = [&](int row, int64_t& o, int64_t& at_lse) {
    const int g = cut.rb * C::kRows + r0 + row;
    const int tok = group_of(p, g), hd = cut.h * p.group + (g - tok * p.group);
    o = cut.b * p.o_sb + static_cast<int64_t>(hd) * p.o_sh + static_cast<int64_t>(tok) * p.o_ss;
    at_lse = (static_cast<int64_t>(cut.b) * p.Hq + hd) * p.T + tok;
  };
  int64_t o, at;
  if (p.lse && warp == 0 && lane < n) {
    place(lane, o, at);
    p.lse[at] = lse_of(m, l);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * (D / 8); i += 256) {
    const int row = i / (D / 8), c = i % (D / 8);
    if (c * 8 >= p.D) continue;
    place(row, o, at);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + o + c * 8) =
        *reinterpret_cast<const uint4*>(tile + row * kStride + c * 8);
  }
}

template <int D>
size_t workspace(int sm_count) {
  return static_cast<size_t>(sm_count) * (2 * Cfg<D>::kRows * (D + 2) * sizeof(float) + sizeof(Cut));
}

template <int D>
cudaError_t launch(AttendParams p, int sm_count, cudaStream_t stream) {
  using C = Cfg<D>;
  auto kern = chunk_kernel<D>;
  static int configured = 0;  // one bit per device ordinal (< 32)
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev >= 32 || !(__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & (1 << dev))) {
    // setmaxnreg.inc would wait forever if the block were launched with fewer registers than
    // the split assumes: check the built register count first.
    cudaFuncAttributes attr;
    if ((err = cudaFuncGetAttributes(&attr, kern)) != cudaSuccess) return err;
    if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidKernelImage;
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (err != cudaSuccess) return err;
    if (dev < 32) __atomic_fetch_or(&configured, 1 << dev, __ATOMIC_ACQ_REL);
  }
  const int64_t rows = static_cast<int64_t>(p.group) * p.T;
  p.row_blocks = static_cast<int>((rows + C::kRows - 1) / C::kRows);
  if (static_cast<int64_t>(p.B) * p.row_blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const int64_t seq_tiles = (static_cast<int64_t>(p.width) * p.page + kTileKeys - 1) / kTileKeys;
  const int64_t most = seq_tiles * p.Hkv * p.row_blocks * p.B;
  const int parts = static_cast<int>(most < sm_count ? most : sm_count);
  const int64_t part_rows = static_cast<int64_t>(sm_count) * 2 * C::kRows;
  p.part_ml = p.part_o + part_rows * D;
  p.cuts = reinterpret_cast<Cut*>(p.part_ml + part_rows * 2);
  err = launch_overlapped(kern, dim3(parts), kThreads, C::kBytes, stream, p);
  if (err != cudaSuccess) return err;
  const int merged = static_cast<int>(rows < C::kRows ? rows : C::kRows);
  return launch_overlapped(merge_kernel<D>, dim3(parts, (merged + 31) / 32), 256, 0, stream, p);
}

}  // namespace
}  // namespace chunk

size_t chunk_workspace_bytes(int D, int sm_count) {
  return D <= 64 ? chunk::workspace<64>(sm_count)
                 : D <= 128 ? chunk::workspace<128>(sm_count) : chunk::workspace<256>(sm_count);
}

cudaError_t launch_chunk(const AttendParams& p, int sm_count, cudaStream_t stream) {
  if (p.D <= 64) return chunk::launch<64>(p, sm_count, stream);
  if (p.D <= 128) return chunk::launch<128>(p, sm_count, stream);
  return chunk::launch<256>(p, sm_count, stream);
}

}  // namespace kv8
}  // namespace ta
