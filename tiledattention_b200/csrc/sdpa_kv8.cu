// Attention of few query rows over the paged 8-bit cache (decoding, checking drafted tokens).
//
//   s_j = scale * (q . k_j) * 2^ek_j          k_j, v_j e4m3 codes, ek_j, ev_j the exponents of
//   o   = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m - ev_j)    their pages' scales,
//   t_j = log2(e) s_j + ev_j                  m a running maximum of t
//
// The value scale joins the exponent: the weights handed to the second product, 2^(t_j - m),
// then measure each key's share of the output in units of its e4m3 codes, so one fp16 weight
// (11 bits, <= 2^8) is right for pages of any scale. The denominator is summed in fp32.
//
// HBM-bound: 2 D bytes a key against 4 D G operations for the G heads that share it. Codes go to
// fp16 in registers (exact; 160 codes/ns/SM measured against the 44 bytes/ns/SM that HBM
// delivers) and feed mma.sync m16n8k16: 16 rows at a time is what decoding has, and a
// tcgen05 tile of 128 rows would be empty for the most part.
//
// One warp = its own keys: it copies kKeys keys a stage with cp.async into its own shared
// memory, keeps its own running maximum, sums and output, and waits for nobody; the four warps
// of a block merge when a (sequence, head) ends. Work is a line of tiles over all sequences
// and heads, cut into equal runs, one a block, so batches of uneven lengths fill the GPU
// evenly; a (sequence, head) that lies in one run is written at once, one that is cut leaves
// partial results for the merge kernel, which starts before this one ends (programmatic
// launch).
//
// Operands without shuffles: K codes are read with 16-byte loads, thread (g, t) of a warp
// taking dims 64 j + 16 t ..+15 of key g, and Q's fragments use the same order of dims. V codes
// come through ldmatrix m16n16.trans.b8, which gives a thread 4 consecutive keys of one dim;
// the keys of score columns are permuted to match (key 16 i + 4 (n / 2) + 2 half + n % 2 for
// column n), so a score fragment is the weight fragment as it stands.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv8.h"
#include "sm100_ptx.cuh"
#include "tiledattention_b200.h"

namespace ta {
namespace kv8 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kGrowth = 8.f;  // log2: the running maximum follows when it grew by more

// NJ: head dim in blocks of 64 (row pitch in shared memory: a power of two). MT: 16-row tiles.
template <int NJ, int MT>
struct Cfg {
  static constexpr int kDim = NJ * 64;
  static constexpr int kPitch = NJ <= 2 ? NJ * 64 : 256;
  static constexpr int kKeys = (NJ <= 2 && MT == 1) ? 32 : 16;  // per warp and stage
  static constexpr int kBlocks = kKeys / 16;
  static constexpr int kTile = kWarps * kKeys;  // keys per block and step
  static constexpr int kRows = 16 * MT;
  static constexpr int kSlot = 2 * kKeys * kPitch;  // K and V bytes of a warp's stage
  // ~96 KB of stages a block, two blocks a SM
  static constexpr int kStages = (96 * 1024) / (kWarps * kSlot) < 6 ? (96 * 1024) / (kWarps * kSlot) : 6;
  // merge: a slot holds kRows x kMergeCols floats
  static constexpr int kMergeCols = kSlot / (kRows * 4) < kDim ? kSlot / (kRows * 4) : kDim;
  static constexpr int kPasses = (kDim + kMergeCols - 1) / kMergeCols;
  static constexpr int kScaleOff = kWarps * kStages * kSlot;
  static constexpr int kScaleBytes = kWarps * kStages * 2 * kBlocks * 4;
  static constexpr int kMlOff = kScaleOff + kScaleBytes;
  static constexpr int kScanOff = kMlOff + 2 * kWarps * kRows * 4;
  static constexpr int kBytes = kScanOff + 64;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
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
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack16(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float pow2f(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Natural-log log-sum-exp of a row from its maximum (log2) and sum; -inf without a key.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (fmaxf(m, -3.4e38f) + log2f(l)) * 0.69314718055994531f;
}

__device__ __forceinline__ SeqExtent extent_of(const AttendParams& p, int b) {
  return checked_extent(p.lengths[b], p.counts ? p.counts[b] : p.T, p.T,
                        static_cast<int64_t>(p.width) * p.page);
}
__device__ __forceinline__ int tiles_of(const SeqExtent& e, int tile) {
  return e.count > 0 ? (e.length + tile - 1) / tile : 0;
}

// Tiles of the whole batch, and those before this thread's share [b0, b1) of it. Called by
// all threads of a block; `report`: record lengths and counts out of range.
struct Scan {
  int64_t total, mine;
};
__device__ __forceinline__ Scan scan_batch(const AttendParams& p, int tile, int64_t per_tile,
                                           int64_t* s_warp, bool report, int& b0, int& b1) {
  const int share = (p.B + blockDim.x - 1) / blockDim.x;
  b0 = min(p.B, static_cast<int>(threadIdx.x) * share);
  b1 = min(p.B, b0 + share);
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) {
    const SeqExtent e = extent_of(p, b);
    if (e.bad && report && p.status) atomicOr(p.status, TA_DEVSTAT_BAD_LENGTH);
    sum += static_cast<int64_t>(tiles_of(e, tile)) * per_tile;
  }
  int64_t incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, d);
    if ((threadIdx.x & 31) >= d) incl += up;
  }
  if ((threadIdx.x & 31) == 31) s_warp[threadIdx.x >> 5] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) before += s_warp[w];
    total += s_warp[w];
  }
  return {total, before + incl - sum};
}

// A place on the line of tiles.
struct Cursor {
  int b, hr, tile, tiles, length;
};

template <int NJ, int MT>
__global__ void __launch_bounds__(kThreads, 2) attend_kernel(const AttendParams p, int d_chunks) {
  using C = Cfg<NJ, MT>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* s_m = reinterpret_cast<float*>(smem + C::kMlOff);
  float* s_l = s_m + kWarps * C::kRows;
  int64_t* s_scan = reinterpret_cast<int64_t*>(smem + C::kScanOff);
  int* s_start = reinterpret_cast<int*>(s_scan + kWarps);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int hrs = p.Hkv * p.row_blocks;

  // Columns beyond the head dim are never copied: they stay zero.
  const bool padded = d_chunks != NJ * 4;
  if (padded)
    for (int i = threadIdx.x; i < C::kScaleOff / 16; i += kThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);

  // This block's run of the line, and the sequence it begins in.
  int b0, b1;
  const Scan sc = scan_batch(p, C::kTile, hrs, s_scan, blockIdx.x == 0, b0, b1);
  const int64_t total = sc.total;
  const int64_t parts = min(static_cast<int64_t>(gridDim.x), total);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x >= parts) return;
  const int64_t w0 = run_begin(blockIdx.x, total, parts);
  const int64_t w1 = run_begin(blockIdx.x + 1, total, parts);
  {
    int64_t at = sc.mine;
    for (int b = b0; b < b1; ++b) {
      const int64_t n = static_cast<int64_t>(tiles_of(extent_of(p, b), C::kTile)) * hrs;
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
    cur.hr = s_start[1] / cur.tiles;
    cur.tile = s_start[1] - cur.hr * cur.tiles;
  }
  Cursor ahead = cur;  // the place of the next copy

  const uint32_t slots = smem_u32(smem) + warp * (C::kStages * C::kSlot);
  const uint32_t scales = smem_u32(smem) + C::kScaleOff + warp * (C::kStages * 2 * C::kBlocks * 4);

  auto advance = [&](Cursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.hr < hrs) return;
    c.hr = 0;
    do {
      if (++c.b >= p.B) return;
      const SeqExtent e = extent_of(p, c.b);
      c.length = e.length;
      c.tiles = tiles_of(e, C::kTile);
    } while (c.tiles == 0);
  };

  // Page ids of this warp's 16-key blocks at `ahead`, fetched one step before their use.
  int page_id[C::kBlocks];
  auto fetch_pages = [&]() {
#pragma unroll
    for (int i = 0; i < C::kBlocks; ++i) {
      const int key = ahead.tile * C::kTile + warp * C::kKeys + i * 16;
      page_id[i] = key < ahead.length
                       ? p.table[ahead.b * p.table_stride + (key >> p.page_shift)] : 0;
    }
  };
  // Starts the copies of this warp's keys at `ahead` into stage st. Rows from the sequence's
  // end on, and blocks with a page id outside the cache, are filled with zeros.
  auto copy_stage = [&](int st) {
    const int h = ahead.hr / p.row_blocks;
    const int key0 = ahead.tile * C::kTile + warp * C::kKeys;
    const uint32_t dst = slots + st * C::kSlot;
#pragma unroll
    for (int i = 0; i < C::kBlocks; ++i) {
      const int key = key0 + i * 16;
      if (key >= ahead.length) continue;
      int id = page_id[i];
      int rows = min(16, ahead.length - key);
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_pages)) {
        if (lane == 0 && p.status) atomicOr(p.status, TA_DEVSTAT_BAD_PAGE);
        id = 0;
        rows = 0;
      }
      const int64_t ph = static_cast<int64_t>(id) * p.Hkv + h;
      const int64_t off = (ph * p.page + (key & (p.page - 1))) * static_cast<int64_t>(p.D);
      const uint8_t* kp = p.pages[0] + off;
      const uint8_t* vp = p.pages[1] + off;
      const int full = rows * d_chunks;  // chunks that exist
      if (!padded) {
#pragma unroll
        for (int c0 = 0; c0 < NJ * 2; ++c0) {
          const int e = c0 * 32 + lane;
          const int row = e / (NJ * 4), c = e % (NJ * 4);
          const uint32_t to = dst + chunk_at<C::kPitch>(i * 16 + row, c);
          const uint32_t n = e < full ? 16u : 0u;
          const int64_t from = n ? e * 16 : 0;
          cp_async16(to, kp + from, n);
          cp_async16(to + C::kKeys * C::kPitch, vp + from, n);
        }
      } else {
        const int recip = (65536 + d_chunks - 1) / d_chunks;  // exact for e < 512
        for (int e = lane; e < 16 * d_chunks; e += 32) {
          const int row = (e * recip) >> 16, c = e - row * d_chunks;
          const uint32_t to = dst + chunk_at<C::kPitch>(i * 16 + row, c);
          const uint32_t n = e < full ? 16u : 0u;
          const int64_t from = n ? e * 16 : 0;
          cp_async16(to, kp + from, n);
          cp_async16(to + C::kKeys * C::kPitch, vp + from, n);
        }
      }
      if (lane < 2) cp_async4(scales + ((st * 2 + lane) * C::kBlocks + i) * 4, p.scale[lane] + ph);
    }
  };

  // ---- the run
  const int64_t steps = w1 - w0;
  fetch_pages();
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) {
    if (s < steps) {
      copy_stage(s);
      if (s + 1 < steps) {
        advance(ahead);
        fetch_pages();
      }
    }
    cp_commit();
  }

  float o[MT][NJ * 8][4];
  float m_run[MT][2], l_run[MT][2], mul[MT][2];
  int lim[MT][2];
  uint32_t qf[MT][NJ][4][4];
  bool fresh = true;
  int begin_tile = cur.tile;
  int st = 0;
  for (int64_t step = 0; step < steps; ++step) {
    cp_wait<C::kStages - 2>();
    __syncwarp();
    {  // the stage freed by the step before is filled again
      const int64_t next = step + C::kStages - 1;
      if (next < steps) {
        copy_stage(st == 0 ? C::kStages - 1 : st - 1);
        if (next + 1 < steps) {
          advance(ahead);
          fetch_pages();
        }
      }
      cp_commit();
    }

    const int h = cur.hr / p.row_blocks, rb = cur.hr - h * p.row_blocks;
    if (fresh) {  // rows of a new (sequence, head): queries, limits, empty sums
      fresh = false;
      begin_tile = cur.tile;
      const SeqExtent e = extent_of(p, cur.b);
      const int rows = p.group * p.T;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int n = 0; n < NJ * 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[mt][n][x] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = rb * C::kRows + mt * 16 + half * 8 + g;
          const int tok = r / p.group, hd = h * p.group + (r - tok * p.group);
          const bool real = r < rows && tok < e.count;
          lim[mt][half] = real ? row_limit(e.length, e.count, tok, p.causal) : 0;
          m_run[mt][half] = -INFINITY;
          l_run[mt][half] = 0.f;
          const uint16_t* q = static_cast<const uint16_t*>(p.q) + cur.b * p.q_sb +
                              static_cast<int64_t>(hd) * p.q_sh + static_cast<int64_t>(tok) * p.q_ss;
          uint32_t w[NJ][8];
          float amax = 0.f;
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const int c = j * 4 + t;  // 16 dims from 16 c
              uint4 x = make_uint4(0, 0, 0, 0);
              if (real && c < d_chunks) x = *reinterpret_cast<const uint4*>(q + c * 16 + v * 8);
              w[j][4 * v] = x.x;
              w[j][4 * v + 1] = x.y;
              w[j][4 * v + 2] = x.z;
              w[j][4 * v + 3] = x.w;
            }
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const float2 a = unpack16(w[j][v], p.bf16);
              amax = fmaxf(amax, fmaxf(fabsf(a.x), fabsf(a.y)));
            }
          }
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          // The row times a power of two, with its largest value in [2^13, 2^14): fp16 then
          // holds every bf16 or fp16 value of the row to 2^-38 of the largest. Held to
          // exponents whose factors are normal float32 values.
          const int ex = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 13, -126), 113);
          const float up = pow2f(-ex);
          mul[mt][half] = p.scale_log2 * pow2f(ex);
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float2 a = unpack16(w[j][2 * v], p.bf16);
              const float2 c = unpack16(w[j][2 * v + 1], p.bf16);
              qf[mt][j][v][half] = pack_f16(a.x * up, a.y * up);
              qf[mt][j][v][2 + half] = pack_f16(c.x * up, c.y * up);
            }
        }
      }
    }

    const int key0 = cur.tile * C::kTile + warp * C::kKeys;
    if (key0 < cur.length) {
      const uint32_t kb = slots + st * C::kSlot;
      const uint32_t vb = kb + C::kKeys * C::kPitch;
      // scores
      float s[MT][2 * C::kBlocks][4];
#pragma unroll
      for (int nt = 0; nt < 2 * C::kBlocks; ++nt) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[mt][nt][x] = 0.f;
        const int row = (nt >> 1) * 16 + key_of_column(g, nt & 1);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint4 kw = lds128(kb + chunk_at<C::kPitch>(row, j * 4 + t));
          const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t f0, f1;
            codes_to_f16(w[v], f0, f1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma16816(s[mt][nt], qf[mt][j][v], f0, f1);
          }
        }
      }
      // t = score * scales + exponent of the value scale; maxima
      float back[C::kBlocks];
#pragma unroll
      for (int i = 0; i < C::kBlocks; ++i) {
        const float ks = lds32(scales + (st * 2 * C::kBlocks + i) * 4);
        const int ev = stored_exponent(__float_as_uint(lds32(scales + ((st * 2 + 1) * C::kBlocks + i) * 4)));
        back[i] = pow2f(-ev);
        const float evf = static_cast<float>(ev);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float c0 = mul[mt][0] * ks, c1 = mul[mt][1] * ks;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int key = key0 + i * 16 + 4 * t + 2 * hf;
            float(&x)[4] = s[mt][2 * i + hf];
            x[0] = key < lim[mt][0] ? fmaf(x[0], c0, evf) : -INFINITY;
            x[1] = key + 1 < lim[mt][0] ? fmaf(x[1], c0, evf) : -INFINITY;
            x[2] = key < lim[mt][1] ? fmaf(x[2], c1, evf) : -INFINITY;
            x[3] = key + 1 < lim[mt][1] ? fmaf(x[3], c1, evf) : -INFINITY;
          }
        }
      }
      float cand[MT][2];
      bool grow = false;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float c = -INFINITY;
#pragma unroll
          for (int nt = 0; nt < 2 * C::kBlocks; ++nt)
            c = fmaxf(c, fmaxf(s[mt][nt][2 * half], s[mt][nt][2 * half + 1]));
          c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 1));
          c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 2));
          cand[mt][half] = c;
          grow |= c > m_run[mt][half] + kGrowth;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float a[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            a[half] = 1.f;
            if (cand[mt][half] > m_run[mt][half] + kGrowth) {
              a[half] = ex2_approx(m_run[mt][half] - cand[mt][half]);  // 0 from -inf
              m_run[mt][half] = cand[mt][half];
              l_run[mt][half] *= a[half];
            }
          }
#pragma unroll
          for (int n = 0; n < NJ * 8; ++n) {
            o[mt][n][0] *= a[0];
            o[mt][n][1] *= a[0];
            o[mt][n][2] *= a[1];
            o[mt][n][3] *= a[1];
          }
        }
      }
      // weights and the second product
#pragma unroll
      for (int i = 0; i < C::kBlocks; ++i) {
        // Blocks from the sequence's end on were not copied: what their stage holds must not
        // meet a weight of zero (0 * NaN).
        if (i > 0 && key0 + i * 16 >= cur.length) break;
        // A key that some row may not see yet (later tokens of the same call) must not reach
        // that row through 0 * NaN either.
        bool later = false;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            later |= lim[mt][half] > 0 && lim[mt][half] < min(cur.length, key0 + i * 16 + 16);
        if (__any_sync(0xffffffffu, later)) {
          bool nan = false;
          for (int e = lane; e < 64 * NJ; e += 32)
            nan |= any_nan(lds128(vb + chunk_at<C::kPitch>(i * 16 + e / (NJ * 4), e % (NJ * 4))));
          if (__any_sync(0xffffffffu, nan)) {
#pragma unroll 1
            for (int key = 0; key < 16; ++key)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < NJ * 8; ++n)
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    const int d = n * 8 + 2 * t + (x & 1);
                    const uint32_t c = lds8(vb + chunk_at<C::kPitch>(i * 16 + key, d >> 4) + (d & 15));
                    if ((c & 0x7fu) == 0x7fu && key0 + i * 16 + key < lim[mt][x >> 1])
                      o[mt][n][x] = __int_as_float(0x7fffffff);
                  }
            __syncwarp();
            for (int e = lane; e < 64 * NJ; e += 32) {
              const uint32_t at = vb + chunk_at<C::kPitch>(i * 16 + e / (NJ * 4), e % (NJ * 4));
              sts128(at, without_nan(lds128(at)));
            }
            __syncwarp();
          }
        }
        uint32_t pf[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float m0 = m_run[mt][0] == -INFINITY ? 0.f : m_run[mt][0];
          const float m1 = m_run[mt][1] == -INFINITY ? 0.f : m_run[mt][1];
          float e[2][4];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float(&x)[4] = s[mt][2 * i + hf];
            e[hf][0] = ex2_approx(x[0] - m0);
            e[hf][1] = ex2_approx(x[1] - m0);
            e[hf][2] = ex2_approx(x[2] - m1);
            e[hf][3] = ex2_approx(x[3] - m1);
            pf[mt][2 * hf] = pack_f16(e[hf][0], e[hf][1]);
            pf[mt][2 * hf + 1] = pack_f16(e[hf][2], e[hf][3]);
          }
          l_run[mt][0] = fmaf((e[0][0] + e[0][1]) + (e[1][0] + e[1][1]), back[i], l_run[mt][0]);
          l_run[mt][1] = fmaf((e[0][2] + e[0][3]) + (e[1][2] + e[1][3]), back[i], l_run[mt][1]);
        }
#pragma unroll
        for (int n = 0; n < NJ * 2; ++n) {  // 32 dims
          uint32_t w[4];
          ldsm_codes_t(vb + chunk_at<C::kPitch>(i * 16 + (lane & 15), n * 2 + (lane >> 4)), w);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t f0, f1;
            codes_to_f16(w[x], f0, f1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma16816(o[mt][n * 4 + x], pf[mt], f0, f1);
          }
        }
      }
    }

    // ---- the end of this (sequence, head) or of the run: merge the warps
    const bool seq_end = cur.tile + 1 == cur.tiles;
    if (seq_end || step + 1 == steps) {
      const bool whole = seq_end && begin_tile == 0;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float l = l_run[mt][half];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          if (t == 0) {
            s_m[warp * C::kRows + mt * 16 + half * 8 + g] = m_run[mt][half];
            s_l[warp * C::kRows + mt * 16 + half * 8 + g] = l;
          }
        }
      __syncthreads();
      float f[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = mt * 16 + half * 8 + g;
          float m = s_m[r];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w * C::kRows + r]);
          f[mt][half] = ex2_approx(m_run[mt][half] - m);  // unused where the maximum is -inf
        }
      // A warp's just-read stage is free until the next step's copies: it takes the warp's
      // output, kMergeCols dims at a time, and all threads add the four.
      float* mine = reinterpret_cast<float*>(smem + (warp * C::kStages + st) * C::kSlot);
      constexpr int kMask = C::kMergeCols / 8 < 8 ? C::kMergeCols / 8 - 1 : 7;
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (begin_tile == 0 ? 1 : 0)) * C::kRows;
#pragma unroll
      for (int pass = 0; pass < C::kPasses; ++pass) {
        if (pass > 0) __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < NJ * 8; ++n) {
            if (n * 8 / C::kMergeCols != pass) continue;
            const int col = n * 8 - pass * C::kMergeCols + 2 * t;
            const int r0 = mt * 16 + g;
            const int x = (r0 & kMask) * 8;  // rows r0 and r0 + 8 alike
            const bool any0 = m_run[mt][0] != -INFINITY, any1 = m_run[mt][1] != -INFINITY;
            *reinterpret_cast<float2*>(mine + r0 * C::kMergeCols + (col ^ x)) =
                make_float2(any0 ? o[mt][n][0] * f[mt][0] : 0.f, any0 ? o[mt][n][1] * f[mt][0] : 0.f);
            *reinterpret_cast<float2*>(mine + (r0 + 8) * C::kMergeCols + (col ^ x)) =
                make_float2(any1 ? o[mt][n][2] * f[mt][1] : 0.f, any1 ? o[mt][n][3] * f[mt][1] : 0.f);
          }
        __syncthreads();
        for (int i = threadIdx.x; i < C::kRows * C::kMergeCols / 4; i += kThreads) {
          const int r = i / (C::kMergeCols / 4), c4 = (i % (C::kMergeCols / 4)) * 4;
          const int d = pass * C::kMergeCols + c4;
          const int row = rb * C::kRows + r;
          if (row >= p.group * p.T || d >= p.D) continue;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w * C::kRows + r]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(
                smem + (w * C::kStages + st) * C::kSlot +
                4 * (r * C::kMergeCols + (c4 ^ ((r & kMask) * 8))));
            a.x += v.x;
            a.y += v.y;
            a.z += v.z;
            a.w += v.w;
            const float mw = s_m[w * C::kRows + r];
            // A sum without a maximum is 0, or NaN where every score was NaN: it is kept.
            l = fmaf(s_l[w * C::kRows + r], mw == -INFINITY ? 1.f : ex2_approx(mw - m), l);
          }
          if (whole) {
            const int tok = row / p.group, hd = h * p.group + (row - tok * p.group);
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
      __syncthreads();
      if (padded) {  // the merge wrote over the zero columns of this warp's stage
        uint4* z = reinterpret_cast<uint4*>(mine);
        for (int i = lane; i < C::kSlot / 16; i += 32) z[i] = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      fresh = true;
    }
    advance(cur);
    st = st + 1 == C::kStages ? 0 : st + 1;
  }
}

// Merges the partial results of (sequence, head)s that several runs share, and writes the rows
// of sequences without keys. One block: kWarps rows, a warp each, or with `spread` one row
// whose runs the warps divide (few rows, many runs).
template <int NJ, int MT>
__global__ void __launch_bounds__(kThreads) merge_kernel(const AttendParams p, int parts_max,
                                                         int spread) {
  using C = Cfg<NJ, MT>;
  constexpr int kVec = NJ <= 2 ? 1 : 2;  // float4 a lane: 32 lanes cover the head dim
  __shared__ int64_t s_scan[kWarps];
  __shared__ float s_o[kWarps][NJ * 64];
  __shared__ float s_ml[kWarps][2];
  __shared__ int64_t s_at;
  __shared__ int s_tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.group * p.T;
  const int per = spread ? 1 : kWarps;
  const int row_groups = (rows + per - 1) / per;
  const int rg = blockIdx.x % row_groups;
  const int h = (blockIdx.x / row_groups) % p.Hkv;
  const int b = blockIdx.x / row_groups / p.Hkv;
  const int hrs = p.Hkv * p.row_blocks;
  int b0, b1;
  const Scan sc = scan_batch(p, C::kTile, hrs, s_scan, false, b0, b1);
  {
    int64_t at = sc.mine;
    for (int i = b0; i < b1; ++i) {
      const int n = tiles_of(extent_of(p, i), C::kTile);
      if (i == b) {
        s_at = at;
        s_tiles = n;
      }
      at += static_cast<int64_t>(n) * hrs;
    }
  }
  __syncthreads();
  const int tiles = s_tiles;
  const int row = spread ? rg : rg * kWarps + warp;
  const int rb = row / C::kRows, r = row - rb * C::kRows;
  const int64_t parts = min(static_cast<int64_t>(parts_max), sc.total);
  int64_t i0 = 0, i1 = 0, first = 0;
  if (tiles > 0) {
    first = s_at + static_cast<int64_t>(h * p.row_blocks + rb) * tiles;
    i0 = run_of(first, sc.total, parts);
    i1 = run_of(first + tiles - 1, sc.total, parts);
  }
  const bool mine = row < rows && !(tiles > 0 && i0 == i1);  // else that run wrote the row
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (spread && !mine) return;  // one row a block: all its threads alike
  float m = -INFINITY, l = 0.f;
  float4 a[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine && tiles > 0) {
    const int64_t step = spread ? kWarps : 1;
#pragma unroll 4
    for (int64_t i = i0 + (spread ? warp : 0); i <= i1; i += step) {
      // a run that begins at or before `first` has this head's first tile: its second slot
      const int second = run_begin(i, sc.total, parts) <= first ? 1 : 0;
      const int64_t at = (i * 2 + second) * C::kRows + r;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
      const float mn = fmaxf(m, ml.x);
      // without a maximum: sums of 0 or NaN and outputs of 0, kept as they are
      const float fa = m == -INFINITY ? 1.f : exp2f(m - mn);
      const float fb = ml.x == -INFINITY ? 1.f : exp2f(ml.x - mn);
      l = l * fa + ml.y * fb;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        const int d = (v * 32 + lane) * 4;
        if (d < p.D) {
          const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * C::kDim + d);
          a[v].x = a[v].x * fa + x.x * fb;
          a[v].y = a[v].y * fa + x.y * fb;
          a[v].z = a[v].z * fa + x.z * fb;
          a[v].w = a[v].w * fa + x.w * fb;
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
  const int tok = row / p.group, hd = h * p.group + (row - tok * p.group);
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

// Rows per block: one 16-row tile while they fit, else (up to head dim 128) two, so that a
// cache read serves 32 rows.
int m_tiles(int rows, int D) { return rows > 16 && D <= 128 ? 2 : 1; }

template <int NJ, int MT>
cudaError_t launch(AttendParams p, int sm_count, cudaStream_t stream) {
  using C = Cfg<NJ, MT>;
  static_assert(C::kStages >= 2, "two stages at least");
  auto kern = attend_kernel<NJ, MT>;
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
  // Most tiles that the lengths can ask for; more blocks than that would have none.
  const int64_t seq_tiles = (static_cast<int64_t>(p.width) * p.page + C::kTile - 1) / C::kTile;
  const int64_t per_seq = seq_tiles * p.Hkv * p.row_blocks;
  if (per_seq > 0x7fffffffll) return cudaErrorInvalidValue;
  const int64_t most = per_seq * p.B;
  const int parts = static_cast<int>(most < 2ll * sm_count ? most : 2ll * sm_count);
  const int64_t part_rows = static_cast<int64_t>(2 * sm_count) * 2 * C::kRows;
  p.part_ml = p.part_o + part_rows * C::kDim;
  kern<<<parts, kThreads, C::kBytes, stream>>>(p, p.D / 16);
  if ((err = cudaGetLastError()) != cudaSuccess) return err;

  const int64_t few = static_cast<int64_t>(p.B) * p.Hkv * rows;
  const int spread = few <= 2ll * sm_count ? 1 : 0;
  const int64_t blocks = spread ? few : static_cast<int64_t>(p.B) * p.Hkv * ((rows + kWarps - 1) / kWarps);
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, merge_kernel<NJ, MT>, p, parts, spread);
}

}  // namespace

size_t attend_workspace_bytes(int, int Hq, int Hkv, int T, int D, int sm_count) {
  const int64_t rows = static_cast<int64_t>(2 * sm_count) * 2 * 16 *
                       m_tiles((Hq / Hkv) * T, D);
  const int dim = (D + 63) / 64 * 64;
  return static_cast<size_t>(rows) * (dim + 2) * sizeof(float);
}

cudaError_t launch_attend(const AttendParams& p, int sm_count, cudaStream_t stream) {
  const int nj = (p.D + 63) / 64;
  const int mt = m_tiles(p.group * p.T, p.D);
  if (mt == 2) return nj == 1 ? launch<1, 2>(p, sm_count, stream) : launch<2, 2>(p, sm_count, stream);
  switch (nj) {
    case 1: return launch<1, 1>(p, sm_count, stream);
    case 2: return launch<2, 1>(p, sm_count, stream);
    case 3: return launch<3, 1>(p, sm_count, stream);
    default: return launch<4, 1>(p, sm_count, stream);
  }
}

}  // namespace kv8
}  // namespace ta
