// Attention of few query rows over the paged 8-bit cache (decoding, checking drafted tokens).
//
//   s_j = scale * (q . k_j) * 2^ek_j          k_j, v_j e4m3 codes, ek_j, ev_j the log2 of
//   o   = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m - ev_j)    their pages' scales,
//   t_j = log2(e) s_j + ev_j                  m a running maximum of t
//
// The value scale joins the exponent: the weights handed to the second product, 2^(t_j - m),
// then measure each key's share of the output in units of its e4m3 codes, so one fp16 weight
// (11 bits, <= 2^8) is right for pages of any scale. The denominator is summed in fp32.
//
// HBM-bound: 2 D bytes a key against 4 D G operations for the G heads that share it. The codes go
// to fp16 in registers (exact) and feed mma.sync m16n8k16 with the KEYS on the 16-side and the
// rows on the 8-side: scores^T = K q^T and o^T += V^T p^T, so 8 heads of a group fill the
// instruction, where rows on the 16-side would leave half of it and of the output registers
// empty. A tcgen05 tile of 128 rows would be empty for the most part; mma.sync on e4m3 itself
// is no faster (it was measured to run as two fp16 ones with the conversions inside).
//
// One warp = its own keys: it copies 32 keys' K and V in turn by TMA into its own ring in shared
// memory, keeps its own reference, sums and output, and waits for nobody; the four warps of a
// block merge when a (sequence, head) ends. Work is a line of tiles over all sequences and
// heads, cut into equal runs, one a block, so batches of uneven lengths fill the GPU evenly; a
// (sequence, head) that lies in one run is written at once, one that is cut leaves partial
// results for the merge kernel, which starts before this one ends (programmatic launch).
//
// Operands: K codes come through ldmatrix, thread (g, t) of a warp taking dims 16 c + 4 t ..+3 of
// key g for chunk c, and q's fragments use the same order of dims. V codes come through ldmatrix
// m16n16.trans.b8, which gives a thread 4 consecutive positions of one dim; the keys of score
// rows are permuted to match (key_at in kv8.h), and movmatrix turns the weights from score rows to
// the second product's columns. With the TMA swizzle neither ldmatrix meets a bank twice.
//
// What bounds the loop next to HBM is instruction issue (2 conversions for 4 codes, 1 MMA for
// 256 codes and 8 rows), so everything a step does not need is kept out of it: masks are applied only
// where a step reaches a row's limit, a page's scales take one multiply-add a score, page ids are fetched
// for up to 32 steps at once, and the reference of a row's weights moves (and is agreed on between
// lanes) only when a score passes it by 2^15.
//
// Measured: 64 sequences of 16384, 64 heads over 8, head dim 128: 347 us, 6.2 TB/s (copying
// alone, without any arithmetic: 335). 32 sequences of up to 4096, 32 heads over 8: 32 us,
// 4.1 TB/s (5 us of it the merge kernel, 5 until the first keys are there). One of 777: 8 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include "kv8_device.cuh"

namespace ta {
namespace kv8 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = kKeysPerStep;  // of a warp: the depth of the second product's MMA
constexpr int kBlocks = kKeys / 16;
// Weights are 2^(t - ref) with ref set to 7 below the row's largest t and moved when t passes
// it by 15: the largest weight then is between 2^7 and 2^15, inside fp16, and what fp16 rounds
// away at its lower end (2^-25) is at most 2^-32 of it.
constexpr float kBelow = 7.f, kGrowth = 15.f;

// NJ: head dim in blocks of 64. NT: tiles of 8 rows.
template <int NJ, int NT>
struct Cfg {
  static constexpr int kDim = NJ * 64;
  static constexpr int kPlanes = NJ <= 2 ? 1 : 2;  // columns of a unit: planes of kCols bytes
  static constexpr int kCols = NJ == 1 ? 64 : 128;
  static constexpr int kTile = kWarps * kKeys;     // keys per block and step
  static constexpr int kRows = 8 * NT;
  static constexpr int kPlane = kKeys * kCols;
  static constexpr int kUnit = kPlanes * kPlane;   // K or V bytes of a warp's step
  // Blocks a SM, as the registers allow (the output takes 16 NJ NT of them, q 8 NJ NT where it
  // is not shared), and the ring's units, as shared memory then allows. One block more costs
  // spills and time: 16 sequences of 8192, 8 heads, head dim 128, 16 rows 91 us with 3 blocks,
  // 66 with 2; head dim 64, 32 rows 101 and 69. <2, 4> and <4, 2> spill with 2 blocks too (338 and 54
  // bytes of stores at 255 registers).
  static constexpr bool kQShared = NJ * NT > 6;
  static constexpr int kBlocksPerSm = NJ * NT == 1 ? 4 : NJ * NT == 2 ? 3 : 2;
  static constexpr int kUnits = NJ == 1 ? 6 : NJ == 2 ? (NT == 1 ? 4 : NT == 2 ? 6 : 5) : 3;
  static constexpr int kScaleSteps = 4;  // steps whose scales are kept: more than units ahead / 2
  // merge: a unit holds kRows x kMergeCols floats
  static constexpr int kMergeCols = kUnit / (kRows * 4) < kDim ? kUnit / (kRows * 4) : kDim;
  static constexpr int kPasses = (kDim + kMergeCols - 1) / kMergeCols;
  static constexpr int kQOff = kWarps * kUnits * kUnit;
  static constexpr int kQBytes = kQShared ? NT * NJ * 2 * 512 : 0;
  static constexpr int kScaleOff = kQOff + kQBytes;
  static constexpr int kScaleBytes = kWarps * kScaleSteps * 2 * kBlocks * 4;
  static constexpr int kMlOff = kScaleOff + kScaleBytes;
  static constexpr int kBarOff = kMlOff + 2 * kWarps * kRows * 4;
  static constexpr int kScanOff = kBarOff + kWarps * kUnits * 8;
  static constexpr int kRowsOff = kScanOff + 64;
  static constexpr int kBytes = kRowsOff + (kQShared ? 2 * kWarps * kRows * 4 : 0) + 1024;  // slack: units are 1024-byte aligned
};
constexpr uint64_t kTimeoutNs = 1000000000ull;  // 1 s per wait for a copy

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float lds32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w) : "memory");
}
// Which bytes of a word are e4m3 NaN (0x7f, 0xff): their top bit.
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ bool any_nan(const uint4& v) {
  return (nan_bits(v.x) | nan_bits(v.y) | nan_bits(v.z) | nan_bits(v.w)) != 0;
}
__device__ __forceinline__ uint4 without_nan(uint4 v) {
  v.x &= ~((nan_bits(v.x) >> 7) * 0xffu);
  v.y &= ~((nan_bits(v.y) >> 7) * 0xffu);
  v.z &= ~((nan_bits(v.z) >> 7) * 0xffu);
  v.w &= ~((nan_bits(v.w) >> 7) * 0xffu);
  return v;
}
// Four matrices of 8 rows x 16 codes: r[m] the codes 4t .. 4t+3 of row g of matrix m.
__device__ __forceinline__ void ldsm_codes(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// 16 keys x 32 dims of codes: r[0], r[1] dims g, g + 8 of the first 16, r[2], r[3] of the second,
// each 4 codes of keys 4t .. 4t+3.
__device__ __forceinline__ void ldsm_codes_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// Four e4m3 codes -> two packed fp16 pairs (exact).
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit values held two a thread.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ int tiles_of(const SeqExtent& e, int tile) {
  return e.count > 0 ? tiles_for(e.length, tile) : 0;
}
// On the line, rows of one (sequence, head) take a unit for each tile, behind kBefore units for their
// queries and their merge. Without these units a run over many short sequences ends last (32
// sequences of up to 4096: 45.8 us); with 1, 2, 3 it is 37.1, 35.0, 34.9 us, and 5 tokens of 8
// sequences at head dim 256 take 39.3, 36.9, 36.9 us.
constexpr int kBefore = 2;
__device__ __forceinline__ int units_of(int tiles) { return tiles > 0 ? tiles + kBefore : 0; }

// A place on the line.
struct Cursor {
  int b, h, rb, tile, tiles, length;
  int left;  // units to the run's end, this tile's included: none without a tile
};

template <int NJ, int NT>
__global__ void __launch_bounds__(kThreads, (Cfg<NJ, NT>::kBlocksPerSm))
    attend_kernel(const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const AttendParams p) {
  using C = Cfg<NJ, NT>;
  constexpr int kU = C::kUnits;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* s_m = reinterpret_cast<float*>(smem + C::kMlOff);
  float* s_l = s_m + kWarps * C::kRows;
  int64_t* s_scan = reinterpret_cast<int64_t*>(smem + C::kScanOff);
  int* s_start = reinterpret_cast<int*>(s_scan + kWarps);
  volatile int* abort_flag = s_start + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff) + warp * kU;
  if (lane == 0) {
    for (int i = 0; i < kU; ++i) mbar_init(full + i, 1);
    fence_mbar_init();
    if (warp == 0) *abort_flag = 0;
  }
  // Launched before the kernel before it has ended (programmatic launch: 2 us of 35 saved in a row of
  // calls): nothing that it may write is read above this line. The merge kernel does not let the
  // next call in before its own end: blocks that came while it ran made a call of 64 sequences
  // of 16384 take 430 us for 350.
  wait_for_stream();

  // This block's run of the line, and the sequence it begins in.
  const int hrs = p.Hkv * p.row_blocks;
  const Scan sc = scan_items<kWarps>(p.B, s_scan, [&](int b) {
    const SeqExtent e = extent_of(p, b);
    report_extent(p, e);
    const int tiles = tiles_of(e, C::kTile);
    if (tiles == 0 && b % gridDim.x == blockIdx.x)  // no run comes by: the merge kernel writes the rows
      for (int i = 0; i < hrs; ++i) p.spans[static_cast<int64_t>(b) * hrs + i] = make_int2(1, 0);
    return static_cast<int64_t>(units_of(tiles)) * hrs;
  });
  const int64_t total = sc.total;
  const int64_t parts = min(static_cast<int64_t>(gridDim.x), total);
  let_next_kernel_in();
  if (blockIdx.x >= parts) return;
  const int64_t w0 = run_begin(blockIdx.x, total, parts), w1 = run_begin(blockIdx.x + 1, total, parts);
  {
    int64_t at = sc.mine;
    for (int b = sc.i0; b < sc.i1; ++b) {
      const int64_t n = static_cast<int64_t>(units_of(tiles_of(extent_of(p, b), C::kTile))) * hrs;
      if (at <= w0 && w0 < at + n) {
        s_start[0] = b;
        s_start[1] = static_cast<int>(w0 - at);  // < 2^31: checked by the launcher
      }
      at += n;
    }
  }
  __syncthreads();

  Cursor cur;
  cur.b = s_start[0];
  {
    const SeqExtent e = extent_of(p, cur.b);
    cur.length = e.length;
    cur.tiles = tiles_of(e, C::kTile);
    const int hr = s_start[1] / units_of(cur.tiles);
    const int at = s_start[1] - hr * units_of(cur.tiles);
    cur.tile = max(0, at - kBefore);
    cur.h = hr / p.row_blocks;
    cur.rb = hr - cur.h * p.row_blocks;
    cur.left = static_cast<int>(w1 - w0) - max(0, kBefore - at);
  }
  if (cur.left <= 0) return;  // a run without a tile
  auto next_rows = [&](Cursor& c) {  // from a tile's end to the next rows with tiles, if any is left
    if (c.left <= 0) return;
    c.left -= kBefore;
    c.tile = 0;
    if (++c.rb < p.row_blocks) return;
    c.rb = 0;
    if (++c.h < p.Hkv) return;
    c.h = 0;
    do {
      if (++c.b >= p.B) return;
      const SeqExtent e = extent_of(p, c.b);
      c.length = e.length;
      c.tiles = tiles_of(e, C::kTile);
    } while (c.tiles == 0);
  };

  // The ring: unit 2 n is K of this warp's keys of step n, unit 2 n + 1 their V. Lane l holds the
  // planes (page, head) of the l-th of up to 32 steps from `ahead` on, fetched at once a step
  // before the first of them; -1: behind the sequence's end, not copied (whole boxes: the rest
  // of its last page comes along); -2: a page outside the cache, not copied, its block marked in
  // `left_out` (4 steps' marks in turn).
  const uint32_t ring = smem_u32(smem) + warp * (kU * C::kUnit);
  const uint32_t scales = smem_u32(smem) + C::kScaleOff + warp * (C::kScaleSteps * 2 * kBlocks * 4);
  const int box = min(p.page, kKeys);
  const int row_at = (warp * kKeys) & (p.page - 1);  // in its page: a tile is whole pages
  const float* scale_of = p.scale[lane & 1];          // lane 2 i + kv copies the scale of block i
  Cursor ahead = cur;
  int held = 0, held_at = 0, held_plane[kBlocks];  // steps in the lanes, the next one to copy
  int plane_at[kBlocks] = {-1, -1};                // of the step copied last
  uint32_t left_out = 0;
  auto fetch_pages = [&]() {  // of the next steps: none at the run's end
    held = max(0, min(min(ahead.tiles - ahead.tile, ahead.left), 32));
    held_at = 0;
    const int32_t* row = p.table + ahead.b * p.table_stride;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const uint32_t key = static_cast<uint32_t>(ahead.tile + lane) * C::kTile + warp * kKeys + i * 16;
      held_plane[i] = -1;
      if (lane < held && key < static_cast<uint32_t>(ahead.length)) {
        const int id = row[key >> p.page_shift];
        const bool good = static_cast<unsigned>(id) < static_cast<unsigned>(p.num_pages);
        held_plane[i] = good ? id * p.Hkv + ahead.h : -2;
        if (!good && p.status) atomicOr(p.status, TA_DEVSTAT_BAD_PAGE);
      }
    }
    ahead.tile += held;
    ahead.left -= held;
  };
  int issue_slot = 0;
  auto copy_unit = [&](const CUtensorMap* map) {
    if (lane == 0) {
      uint64_t* bar = full + issue_slot;
      const uint32_t dst = ring + issue_slot * C::kUnit;
      const bool first = plane_at[0] >= 0, second = box < kKeys && plane_at[1] >= 0;
      mbar_arrive_expect_tx(bar, (first + second) * box * (C::kPlanes * C::kCols));
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
        if (i == 0 ? first : second)
#pragma unroll
          for (int c = 0; c < C::kPlanes; ++c)
            tma_load_3d(dst + c * C::kPlane + i * 16 * C::kCols, map, bar, c * 128, row_at, plane_at[i]);
    }
    issue_slot = issue_slot + 1 == kU ? 0 : issue_slot + 1;
  };
  bool copied_k = false;  // the copies of V follow those of K
  auto copy_k = [&](int n) {
    copied_k = held_at < held;
    if (copied_k) {
      const int slot4 = n & 3;
      left_out &= ~(((1u << kBlocks) - 1) << (slot4 * kBlocks));
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        plane_at[i] = __shfl_sync(0xffffffffu, held_plane[i], held_at);
        if (plane_at[i] == -2) left_out |= 1u << (slot4 * kBlocks + i);
      }
      const int mine = lane < 2 ? plane_at[0] : plane_at[1];
      if (lane < 2 * kBlocks && mine >= 0)
        cp_async4(scales + ((slot4 * 2 + (lane & 1)) * kBlocks + (lane >> 1)) * 4, scale_of + mine);
      copy_unit(&map_k);
      if (++held_at == held) {
        if (ahead.tile == ahead.tiles) next_rows(ahead);
        fetch_pages();
      }
    }
    cp_commit();
  };
  auto copy_v = [&]() {
    if (copied_k) copy_unit(&map_v);
  };
  fetch_pages();

  int slot = 0;
  uint32_t parity = 0;
  auto wait_unit = [&]() {
    if (!mbar_wait_bounded(full + slot, parity, abort_flag, kTimeoutNs) && lane == 0 &&
        !*abort_flag) {
      *abort_flag = 1;
      if (p.status) atomicOr(p.status, TA_DEVSTAT_TIMEOUT_LOAD);
    }
    __syncwarp();  // also: every lane is done with the unit before, which is filled again now
  };
  auto next_unit = [&]() {
    if (++slot == kU) {
      slot = 0;
      parity ^= 1;
    }
  };

  // Of 8-row tile nt a thread holds rows 2t and 2t + 1 of scores and output, row g of q.
  float o[NJ * 4][NT][4];  // 16 dims: (g, 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)
  float ref[NT][2], l_run[NT][2];
  // A row's factor of the scores and its limit: in registers, or where q is shared in shared memory
  // (a copy for each warp).
  float mul[C::kQShared ? 1 : NT][2];
  int lim[C::kQShared ? 1 : NT][2];
  float* s_mul = reinterpret_cast<float*>(smem + C::kRowsOff) + warp * C::kRows;
  int* s_lim = reinterpret_cast<int*>(smem + C::kRowsOff) + (kWarps + warp) * C::kRows;
  auto factors = [&](int nt) {
    if constexpr (C::kQShared) return *reinterpret_cast<const float2*>(s_mul + nt * 8 + 2 * t);
    else return make_float2(mul[nt][0], mul[nt][1]);
  };
  auto limit_of = [&](int nt, int r) {
    if constexpr (C::kQShared) return s_lim[nt * 8 + 2 * t + r];
    else return lim[nt][r];
  };
  uint32_t qf[C::kQShared ? 1 : NT][NJ * 4][2];  // chunk, pair of dims
  uint4* s_q = reinterpret_cast<uint4*>(smem + C::kQOff);
  int safe = 0;  // keys that every row with any keys sees
  bool fresh = true;
  int steps = 0;
  int begin_tile = cur.tile;
  // Unit u + kU - 1 is copied when unit u is waited for, so kU / 2 steps without work come first.
  for (int step = -(kU / 2);; ++step) {
    if (step >= 0 && fresh) {  // rows of a new (sequence, head): queries, limits, empty sums
      fresh = false;
      begin_tile = cur.tile;
      const SeqExtent e = extent_of(p, cur.b);
      const int rows = p.group * p.T;
      int least = 0x7fffffff;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int m = 0; m < NJ * 4; ++m)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[m][nt][x] = 0.f;
        const int r = cur.rb * C::kRows + nt * 8 + g;
        const int tok = group_of(p, r), hd = cur.h * p.group + (r - tok * p.group);
        const bool real = r < rows && tok < e.count;
        const int limit = real ? row_limit(e.length, e.count, tok, p.causal) : 0;
        if (limit > 0) least = min(least, limit);
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + cur.b * p.q_sb +
                            static_cast<int64_t>(hd) * p.q_sh + static_cast<int64_t>(tok) * p.q_ss;
        uint2 w[NJ * 4];
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < NJ * 4; ++c) {
          w[c] = make_uint2(0, 0);
          if (real && c * 16 < p.D) w[c] = *reinterpret_cast<const uint2*>(q + c * 16 + t * 4);
        }
#pragma unroll
        for (int c = 0; c < NJ * 4; ++c) {
          const float2 a = unpack16(w[c].x, p.bf16), b = unpack16(w[c].y, p.bf16);
          amax = fmaxf(fmaxf(amax, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // The row times a power of two, with its largest value in [2^14, 2^15): fp16 then holds
        // every bf16 or fp16 value of the row to 2^-39 of the largest. Held to exponents whose
        // factors are normal float32 values.
        const int ex = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 14, -126), 113);
        const float up = row_factor(amax, ex), factor = p.scale_log2 * pow2f(ex);
        uint32_t f[NJ * 4][2];
#pragma unroll
        for (int c = 0; c < NJ * 4; ++c) {
          const float2 a = unpack16(w[c].x, p.bf16), b = unpack16(w[c].y, p.bf16);
          f[c][0] = pack_f16(a.x * up, a.y * up);
          f[c][1] = pack_f16(b.x * up, b.y * up);
        }
        if constexpr (C::kQShared) {  // one copy for the block
#pragma unroll
          for (int c = 0; c < NJ * 4; c += 2)
            if (c / 2 % kWarps == warp)
              s_q[(nt * NJ * 2 + c / 2) * 32 + lane] =
                  make_uint4(f[c][0], f[c][1], f[c + 1][0], f[c + 1][1]);
        } else {
#pragma unroll
          for (int c = 0; c < NJ * 4; ++c) {
            qf[nt][c][0] = f[c][0];
            qf[nt][c][1] = f[c][1];
          }
        }
        if constexpr (C::kQShared) {
          if (t == 0) {
            s_mul[nt * 8 + g] = factor;
            s_lim[nt * 8 + g] = limit;
          }
        }
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          if constexpr (!C::kQShared) {  // from row g's lanes to those of columns 2t, 2t + 1
            lim[nt][r2] = __shfl_sync(0xffffffffu, limit, (2 * t + r2) * 4);
            mul[nt][r2] = __shfl_sync(0xffffffffu, factor, (2 * t + r2) * 4);
          }
          ref[nt][r2] = -INFINITY;
          l_run[nt][r2] = 0.f;
        }
      }
      safe = __reduce_min_sync(0xffffffffu, least);
      if constexpr (C::kQShared) __syncthreads();
    }
    if (step >= 0) wait_unit();
    if (kU % 2 == 1) copy_k(step + kU / 2);  // unit 2 step + kU - 1
    else copy_v();
    if (step < 0) {
      if (kU % 2 == 1) copy_v();
      else copy_k(step + kU / 2);
      continue;
    }
    cp_wait<(kU - 1) / 2>();
    __syncwarp();

    const int key0 = cur.tile * C::kTile + warp * kKeys;
    const bool any = key0 < cur.length;
    float s[kBlocks][NT][4];  // keys (set 0, g) and (set 1, g) by rows 2t, 2t + 1
    if (any) {
      const uint32_t kb = ring + slot * C::kUnit;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[i][nt][x] = 0.f;
#pragma unroll
      for (int c = 0; c < NJ * 4; c += 2) {
        uint4 qc[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (C::kQShared) qc[nt] = s_q[(nt * NJ * 2 + c / 2) * 32 + lane];
          else qc[nt] = make_uint4(qf[nt][c][0], qf[nt][c][1], qf[nt][c + 1][0], qf[nt][c + 1][1]);
        }
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          uint32_t w[4];  // (set 0, chunk c), (set 1, c), (set 0, c + 1), (set 1, c + 1)
          ldsm_codes(kb + chunk_at<C::kCols, C::kPlane>(
                              i * 16 + key_of_column(lane & 7, (lane >> 3) & 1), c + (lane >> 4)), w);
          uint32_t a[4][2];
#pragma unroll
          for (int x = 0; x < 4; ++x) codes_to_f16(w[x], a[x][0], a[x][1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(s[i][nt], a[0][0], a[1][0], a[0][1], a[1][1], qc[nt].x, qc[nt].y);
            mma16816(s[i][nt], a[2][0], a[3][0], a[2][1], a[3][1], qc[nt].z, qc[nt].w);
          }
        }
      }
    }
    next_unit();

    uint32_t pf[kBlocks][NT][2];  // weights as the second product's B: set 0, set 1
    if (any) {
      // t = score * c + ev in the scores' place, by the scales of the block's page
      float back[kBlocks];
      const uint32_t marks = left_out >> ((step & 3) * kBlocks) & ((1u << kBlocks) - 1);
      const bool masked = key0 > safe - kKeys || marks;  // some row's limit, or pages to leave out
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint32_t at = scales + ((step & 3) * 2 * kBlocks + i) * 4;
        const float ks = lds32(at);
        const ValueScale vs = value_scale(__float_as_uint(lds32(at + kBlocks * 4)));
        const float e = vs.e;
        back[i] = vs.back;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 f = factors(nt);
          const float c0 = f.x * ks, c1 = f.y * ks;
          s[i][nt][0] = fmaf(s[i][nt][0], c0, e);
          s[i][nt][1] = fmaf(s[i][nt][1], c1, e);
          s[i][nt][2] = fmaf(s[i][nt][2], c0, e);
          s[i][nt][3] = fmaf(s[i][nt][3], c1, e);
        }
        if (masked) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int key = marks >> i & 1 ? 0x7fffffff : key0 + i * 16 + key_of_column(g, x >> 1);
              if (key >= limit_of(nt, x & 1)) s[i][nt][x] = -INFINITY;
            }
        }
      }
      float cand[NT][2];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float m = -INFINITY;
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) m = fmaxf(m, fmaxf(s[i][nt][r], s[i][nt][2 + r]));
          cand[nt][r] = m;
          grow |= m - ref[nt][r] > kGrowth;  // not m > ref + kGrowth, a sum that rounds up from 2^24 on
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float a[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float m = cand[nt][r];  // over the row's keys: the lanes of one t
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            a[r] = 1.f;
            if (m - ref[nt][r] > kGrowth) {
              const float to = m - kBelow;
              a[r] = ex2_approx(ref[nt][r] - to);  // 0 from -inf
              ref[nt][r] = to;
              l_run[nt][r] *= a[r];
            }
          }
#pragma unroll
          for (int m = 0; m < NJ * 4; ++m) {
            o[m][nt][0] *= a[0];
            o[m][nt][1] *= a[1];
            o[m][nt][2] *= a[0];
            o[m][nt][3] *= a[1];
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = ref[nt][0] == -INFINITY ? 0.f : ref[nt][0];
        const float r1 = ref[nt][1] == -INFINITY ? 0.f : ref[nt][1];
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          const float(&x)[4] = s[i][nt];
          const float w0 = ex2_approx(x[0] - r0);
          const float w1 = ex2_approx(x[1] - r1);
          const float w2 = ex2_approx(x[2] - r0);
          const float w3 = ex2_approx(x[3] - r1);
          l_run[nt][0] = fmaf(w0 + w2, back[i], l_run[nt][0]);
          l_run[nt][1] = fmaf(w1 + w3, back[i], l_run[nt][1]);
          pf[i][nt][0] = transpose8(pack_f16(w0, w1));
          pf[i][nt][1] = transpose8(pack_f16(w2, w3));
        }
      }
    }

    wait_unit();
    if (kU % 2 == 1) copy_v();  // unit 2 step + 1 + kU - 1
    else copy_k(step + kU / 2);
    if (any) {
      const uint32_t vb = ring + slot * C::kUnit;
      // What a stage holds must not meet a weight of zero where it may be NaN (0 * NaN): blocks
      // that were not copied, and keys that some row does not see (the rest of the last page,
      // later tokens of the same call).
      const uint32_t marks = left_out >> ((step & 3) * kBlocks) & ((1u << kBlocks) - 1);
      if (key0 > safe - kKeys || marks) {
#pragma unroll 1
        for (int i = 0; i < kBlocks; ++i) {
          const bool copied = key0 + i * 16 < cur.length && !(marks >> i & 1);
          bool nan = !copied;
          if (copied && key0 + i * 16 > safe - 16)
            for (int x = lane; x < 64 * NJ; x += 32)
              nan |= any_nan(lds128(vb + chunk_at<C::kCols, C::kPlane>(i * 16 + x / (NJ * 4), x % (NJ * 4))));
          if (!__any_sync(0xffffffffu, nan)) continue;
          if (copied) {
#pragma unroll 1
            for (int key = 0; key < 16; ++key)
#pragma unroll
              for (int m = 0; m < NJ * 4; ++m)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                  const uint32_t code =
                      lds8(vb + chunk_at<C::kCols, C::kPlane>(i * 16 + key, m) + g + 8 * hi);
                  if ((code & 0x7fu) != 0x7fu) continue;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                      if (key0 + i * 16 + key < limit_of(nt, r))
                        o[m][nt][2 * hi + r] = __int_as_float(0x7fffffff);
                }
            __syncwarp();
          }
          for (int x = lane; x < 64 * NJ; x += 32) {
            const uint32_t at = vb + chunk_at<C::kCols, C::kPlane>(i * 16 + x / (NJ * 4), x % (NJ * 4));
            sts128(at, copied ? without_nan(lds128(at)) : make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_shared();  // before the next copy into this unit
          __syncwarp();
        }
      }
#pragma unroll
      for (int n = 0; n < NJ * 2; ++n)  // 32 dims
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          uint32_t w[4];
          ldsm_codes_t(vb + chunk_at<C::kCols, C::kPlane>(i * 16 + key_at(lane & 15), n * 2 + (lane >> 4)),
                       w);
          uint32_t a[4][2];
#pragma unroll
          for (int x = 0; x < 4; ++x) codes_to_f16(w[x], a[x][0], a[x][1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(o[2 * n][nt], a[0][0], a[1][0], a[0][1], a[1][1], pf[i][nt][0], pf[i][nt][1]);
            mma16816(o[2 * n + 1][nt], a[2][0], a[3][0], a[2][1], a[3][1], pf[i][nt][0], pf[i][nt][1]);
          }
        }
    }

    // ---- the end of this (sequence, head) or of the run: merge the warps
    const bool seq_end = cur.tile + 1 == cur.tiles;
    if (seq_end || cur.left == 1) {
      const bool whole = seq_end && begin_tile == 0;
      if (begin_tile == 0 && threadIdx.x == 0) {  // the runs with parts of these rows
        const int64_t last = w1 - cur.left - cur.tile + cur.tiles - 1;
        p.spans[(static_cast<int64_t>(cur.b) * p.Hkv + cur.h) * p.row_blocks + cur.rb] =
            make_int2(blockIdx.x, whole ? blockIdx.x : static_cast<int>(run_of(last, total, parts)));
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (limit_of(nt, r) == 0) {  // a row without keys: its unmasked scores were of no row
            ref[nt][r] = -INFINITY;
            l_run[nt][r] = 0.f;
          }
          float l = l_run[nt][r];
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          l += __shfl_xor_sync(0xffffffffu, l, 8);
          l += __shfl_xor_sync(0xffffffffu, l, 16);
          if (g == 0) {
            s_m[warp * C::kRows + nt * 8 + 2 * t + r] = ref[nt][r];
            s_l[warp * C::kRows + nt * 8 + 2 * t + r] = l;
          }
        }
      __syncthreads();
      float f[NT][2];  // the warp's share of a row; outputs without a reference are none
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float m = s_m[nt * 8 + 2 * t + r];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w * C::kRows + nt * 8 + 2 * t + r]);
          f[nt][r] = ex2_approx(ref[nt][r] - m);
        }
      // A warp's just-read unit is free until the next step's copies: it takes the warp's
      // output, kMergeCols dims at a time, and all threads add the four.
      float* mine = reinterpret_cast<float*>(smem + (warp * kU + slot) * C::kUnit);
      constexpr int kMask = C::kMergeCols / 8 < 4 ? C::kMergeCols / 8 - 1 : 3;  // banks: see below
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (begin_tile == 0 ? 1 : 0)) * C::kRows;
#pragma unroll
      for (int pass = 0; pass < C::kPasses; ++pass) {
        if (pass > 0) __syncthreads();
#pragma unroll
        for (int m = 0; m < NJ * 8; ++m) {  // 8 dims
          if (m * 8 / C::kMergeCols != pass) continue;
          const int col = (m * 8 - pass * C::kMergeCols + g) ^ ((t & kMask) * 8);  // t: row / 2
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              mine[(nt * 8 + 2 * t + r) * C::kMergeCols + col] =
                  ref[nt][r] != -INFINITY ? o[m / 2][nt][2 * (m & 1) + r] * f[nt][r] : 0.f;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C::kRows * C::kMergeCols / 4; i += kThreads) {
          const int r = i / (C::kMergeCols / 4), c4 = (i % (C::kMergeCols / 4)) * 4;
          const int d = pass * C::kMergeCols + c4;
          const int row = cur.rb * C::kRows + r;
          if (row >= p.group * p.T || d >= p.D) continue;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w * C::kRows + r]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(
                smem + (w * kU + slot) * C::kUnit +
                4 * (r * C::kMergeCols + (c4 ^ (((r >> 1) & kMask) * 8))));
            a.x += v.x;
            a.y += v.y;
            a.z += v.z;
            a.w += v.w;
            const float mw = s_m[w * C::kRows + r];
            // A sum without a reference is 0, or NaN where every score was NaN: it is kept.
            l = fmaf(s_l[w * C::kRows + r], mw == -INFINITY ? 1.f : ex2_approx(mw - m), l);
          }
          if (whole) {
            const int tok = group_of(p, row), hd = cur.h * p.group + (row - tok * p.group);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            uint16_t* out = static_cast<uint16_t*>(p.o) + cur.b * p.o_sb + hd * p.o_sh + tok * p.o_ss + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(pack16(a.x * inv, a.y * inv, p.bf16),
                                                        pack16(a.z * inv, a.w * inv, p.bf16));
            if (p.lse && d == 0)
              p.lse[(static_cast<int64_t>(cur.b) * p.Hq + hd) * p.T + tok] = lse_of(m, l);
          } else {
            *reinterpret_cast<float4*>(p.part_o + (part + r) * C::kDim + d) = a;
            if (d == 0)
              *reinterpret_cast<float2*>(p.part_ml + (part + r) * 2) = make_float2(m, l);
          }
        }
      }
      fence_proxy_async_shared();  // before the next copy into this unit
      __syncthreads();
      fresh = true;
    }
    next_unit();
    --cur.left;
    if (seq_end) next_rows(cur);
    else ++cur.tile;
    ++steps;
    if (cur.left <= 0) break;
  }
  if (*abort_flag) {  // a copy was late: every issued one must land before the block ends
    volatile int no_abort = 0;
    for (int u = max(0, 2 * steps - kU); u < 2 * steps; ++u)
      if (!mbar_wait_bounded(full + u % kU, (u / kU) & 1, &no_abort, kTimeoutNs) && lane == 0 &&
          p.status)
        atomicOr(p.status, TA_DEVSTAT_TIMEOUT_DRAIN);
  }
}

// Merges the partial results of (sequence, head)s that several runs share, and writes the rows
// of sequences without keys: both by the attend kernel's records, and nothing of it is read before
// that kernel has ended (lengths read earlier, while it runs, would save 0.4 us of 32). One block: kWarps
// rows, a warp each, or with `spread` one row whose runs the warps divide (few rows, many runs).
template <int NJ, int NT>
__global__ void __launch_bounds__(kThreads) merge_kernel(const AttendParams p, int parts, int spread) {
  using C = Cfg<NJ, NT>;
  constexpr int kVec = NJ <= 2 ? 1 : 2;  // float4 a lane: 32 lanes cover the head dim
  __shared__ float s_o[kWarps][NJ * 64];
  __shared__ float s_ml[kWarps][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.group * p.T;
  const int per = spread ? 1 : kWarps;
  const int row_groups = (rows + per - 1) / per;
  const int bh = blockIdx.x / row_groups;
  const int rg = blockIdx.x - bh * row_groups;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int row = spread ? rg : rg * kWarps + warp;
  const int rb = row / C::kRows, r = row - rb * C::kRows;
  wait_for_stream();
  int i0 = 0, i1 = 0;
  if (row < rows) {
    const int2 span = p.spans[static_cast<int64_t>(bh) * p.row_blocks + rb];
    i0 = max(span.x, 0);
    i1 = min(span.y, parts - 1);
  }
  const bool mine = i0 != i1;  // else one run wrote the row; i0 > i1: no run has a key of it
  if (spread && !mine) return;  // one row a block: all its threads alike
  float m = -INFINITY, l = 0.f;
  float4 a[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i0 < i1) {
    const int step = spread ? kWarps : 1;
    constexpr int kAtOnce = 4;  // parts whose loads are in flight together
    for (int i = i0 + (spread ? warp : 0); i <= i1; i += kAtOnce * step) {
      float2 ml[kAtOnce];
      float4 x[kAtOnce][kVec];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int run = i + k * step;
        ml[k] = make_float2(-INFINITY, 0.f);  // no part: a sum and outputs of 0
        // the run with this head's first tile left its part in its second slot
        const int64_t at = (static_cast<int64_t>(run) * 2 + (run == i0 ? 1 : 0)) * C::kRows + r;
        if (run <= i1) ml[k] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          const int d = (v * 32 + lane) * 4;
          x[k][v] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (run <= i1 && d < p.D) x[k][v] = *reinterpret_cast<const float4*>(p.part_o + at * C::kDim + d);
        }
      }
      float mn = m;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, ml[k].x);
      // without a maximum: sums of 0 or NaN and outputs of 0, kept as they are
      const float fa = m == -INFINITY ? 1.f : exp2f(m - mn);
      l *= fa;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        a[v].x *= fa;
        a[v].y *= fa;
        a[v].z *= fa;
        a[v].w *= fa;
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float fb = ml[k].x == -INFINITY ? 1.f : exp2f(ml[k].x - mn);
        l = fmaf(ml[k].y, fb, l);
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          a[v].x = fmaf(x[k][v].x, fb, a[v].x);
          a[v].y = fmaf(x[k][v].y, fb, a[v].y);
          a[v].z = fmaf(x[k][v].z, fb, a[v].z);
          a[v].w = fmaf(x[k][v].w, fb, a[v].w);
        }
      }
      m = mn;
    }
  }
  if (spread) {
    if (lane == 0) {
      s_ml[warp][0] = m;
      s_ml[warp][1] = l;
    }
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int d = (v * 32 + lane) * 4;
      if (d < NJ * 64) *reinterpret_cast<float4*>(&s_o[warp][d]) = a[v];
    }
    __syncthreads();
    if (warp != 0) return;
    m = fmaxf(fmaxf(s_ml[0][0], s_ml[1][0]), fmaxf(s_ml[2][0], s_ml[3][0]));
    l = 0.f;
#pragma unroll
    for (int v = 0; v < kVec; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_ml[w][0] == -INFINITY ? 1.f : exp2f(s_ml[w][0] - m);
      l = fmaf(s_ml[w][1], f, l);
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        const int d = (v * 32 + lane) * 4;
        if (d < NJ * 64) {
          const float4 x = *reinterpret_cast<const float4*>(&s_o[w][d]);
          a[v].x = fmaf(x.x, f, a[v].x);
          a[v].y = fmaf(x.y, f, a[v].y);
          a[v].z = fmaf(x.z, f, a[v].z);
          a[v].w = fmaf(x.w, f, a[v].w);
        }
      }
    }
  }
  if (!mine) return;
  const int tok = group_of(p, row), hd = h * p.group + (row - tok * p.group);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = static_cast<uint16_t*>(p.o) + b * p.o_sb + hd * p.o_sh + tok * p.o_ss;
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const int d = (v * 32 + lane) * 4;
    if (d < p.D)
      *reinterpret_cast<uint2*>(out + d) = make_uint2(pack16(a[v].x * inv, a[v].y * inv, p.bf16),
                                                      pack16(a[v].z * inv, a[v].w * inv, p.bf16));
  }
  if (p.lse && lane == 0)
    p.lse[(static_cast<int64_t>(b) * p.Hq + hd) * p.T + tok] = lse_of(m, l);
}

template <int NJ, int NT>
cudaError_t launch(AttendParams p, const CUtensorMap& map_k, const CUtensorMap& map_v, int sm_count,
                   cudaStream_t stream) {
  using C = Cfg<NJ, NT>;
  static_assert(C::kUnits >= 3 && (C::kUnits - 1) / 2 + 1 < C::kScaleSteps, "ring and scales");
  auto kern = attend_kernel<NJ, NT>;
  static int configured = 0;  // one bit per device ordinal (< 32)
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev >= 32 || !(__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & (1 << dev))) {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (err != cudaSuccess) return err;
    if (dev < 32) __atomic_fetch_or(&configured, 1 << dev, __ATOMIC_ACQ_REL);
  }
  const int rows = p.group * p.T;
  p.row_blocks = (rows + C::kRows - 1) / C::kRows;
  // Most units that the lengths can ask for; more blocks than that would have none.
  const int64_t seq_tiles = (static_cast<int64_t>(p.width) * p.page + C::kTile - 1) / C::kTile;
  const int64_t per_seq = (seq_tiles + kBefore) * p.Hkv * p.row_blocks;
  if (per_seq > 0x7fffffffll) return cudaErrorInvalidValue;
  const int64_t most = per_seq * p.B;
  const int64_t resident = static_cast<int64_t>(C::kBlocksPerSm) * sm_count;
  const int parts = static_cast<int>(most < resident ? most : resident);
  const int64_t part_rows = resident * 2 * C::kRows;
  p.part_ml = p.part_o + part_rows * C::kDim;
  p.spans = reinterpret_cast<int2*>(p.part_ml + part_rows * 2);
  err = launch_overlapped(kern, dim3(static_cast<unsigned>(parts)), kThreads, C::kBytes, stream, map_k,
                          map_v, p);
  if (err != cudaSuccess) return err;

  const int64_t few = static_cast<int64_t>(p.B) * p.Hkv * rows;
  const int spread = few <= 2ll * sm_count ? 1 : 0;
  const int64_t blocks = spread ? few : static_cast<int64_t>(p.B) * p.Hkv * ((rows + kWarps - 1) / kWarps);
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  return launch_overlapped(merge_kernel<NJ, NT>, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream,
                           p, parts, spread);
}

// One configuration, as an argument.
template <int NJ, int NT>
struct Shape {
  using Config = Cfg<NJ, NT>;
  static cudaError_t launch(const AttendParams& p, const CUtensorMap& k, const CUtensorMap& v, int sms,
                            cudaStream_t stream) {
    return kv8::launch<NJ, NT>(p, k, v, sms, stream);
  }
};

// Calls f with the configuration that serves `rows` rows of head dim D: up to 8 rows one tile, up to
// 16 two, more four while the head dim leaves registers for them, so that a cache read serves
// 32 rows.
template <class F>
auto with_config(int rows, int D, F f) {
  const int nj = (D + 63) / 64;
  if (rows <= 8) {
    if (nj == 1) return f(Shape<1, 1>());
    if (nj == 2) return f(Shape<2, 1>());
    if (nj == 3) return f(Shape<3, 1>());
    return f(Shape<4, 1>());
  }
  if (rows > 16 && nj == 1) return f(Shape<1, 4>());
  if (rows > 16 && nj == 2) return f(Shape<2, 4>());
  if (nj == 1) return f(Shape<1, 2>());
  if (nj == 2) return f(Shape<2, 2>());
  if (nj == 3) return f(Shape<3, 2>());
  return f(Shape<4, 2>());
}

}  // namespace

size_t attend_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int sm_count) {
  const int rows = (Hq / Hkv) * T;
  return with_config(rows, D, [&](auto shape) {
    using C = typename decltype(shape)::Config;
    const size_t row_blocks = (rows + C::kRows - 1) / C::kRows;
    return static_cast<size_t>(C::kBlocksPerSm) * sm_count * 2 * C::kRows * (C::kDim + 2) * sizeof(float) +
           static_cast<size_t>(B) * Hkv * row_blocks * sizeof(int2);
  });
}

cudaError_t launch_attend(const AttendParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                          int sm_count, cudaStream_t stream) {
  return with_config(p.group * p.T, p.D, [&](auto shape) {
    return decltype(shape)::launch(p, map_k, map_v, sm_count, stream);
  });
}

}  // namespace kv8
}  // namespace ta
