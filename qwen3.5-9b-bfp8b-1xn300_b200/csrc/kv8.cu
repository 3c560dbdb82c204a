// kv8.cu — the 8-bit paged KV cache: quantising write, read, and the decode
// attention over it (include/qkv8.h).
//
// Layout.  A page is [kv head][4 blocks]; a block of 16 tokens is 16 bytes of
// scales (K, V, unused), 16 * D bytes of K codes, 16 * D bytes of V codes.
// Codes are stored offset by 128.  The codes of a block stand in the order in
// which the lanes of a warp read them as matrix operands: 512 bytes (16 a lane)
// for every 32 dims, lane 4g + t holding
//   K: tokens rho(g) and rho(g) + 2 (rho(g) = 4 (g / 2) + g % 2), dims 4t .. 4t+3
//      of the first 16 dims, then of the second
//   V: tokens 4t .. 4t+3, dims g and g + 8 of the first 16 dims, then of the second
// so that a lane's four bytes of one token (K) or of one dim (V) are contiguous.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include <cuda_fp16.h>

#include "../../include/qkv8.h"
#include "caller_buffers.h"
#include "common.cuh"
#include "kernels.h"

namespace qc {
namespace {

constexpr int BT = QC_KV8_BLOCK;
constexpr int PAGE_BLOCKS = QC_PAGE / BT;
constexpr int HEAD_BYTES = 16;  // a block's scales

__host__ __device__ constexpr int block_bytes(int dim) { return HEAD_BYTES + 2 * BT * dim; }

// First error of these kernels on this device since the last qc_kv8_check, and the one
// that a check took away: in one step, so that none recorded meanwhile is lost.
__device__ int g_kv8_error, g_kv8_taken;

__global__ void kv8_take_error_kernel() { g_kv8_taken = atomicExch(&g_kv8_error, 0); }

__device__ __forceinline__ int64_t blocks_touched(int64_t pos, int64_t cnt) {
  return cnt > 0 ? (pos + cnt - 1) / BT - pos / BT + 1 : 0;
}

// The smallest power of two s with amax <= 127 s, at least 2^-126.  With amax =
// 1.M * 2^(E - 127) that is 2^(E - 133), or twice it when 1.M > 127 / 64.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = int(u >> 23) - 133 + ((u & 0x7fffffu) > 0x7e0000u);
  e = max(e, -126);
  return __uint_as_float(uint32_t(e + 127) << 23);
}

struct Kv8RowsArgs {
  uint8_t* pool;
  const int32_t *table, *pos, *start;  // start null: one row each
  uint16_t *k, *v;
  int64_t k_ld, v_ld;
  int32_t n_pages, pt_stride, kv_heads, n, rows;
};

// ------------------------------------------------- blocks of many sequences

// Quotient of two counts, in 32 bits where they fit: the 64-bit division is long.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? int64_t(uint32_t(x) / uint32_t(y)) : x / y;
}

// Blocks of the sequences before this thread's run of them, and of all.  The
// sequences are dealt to the CTA's threads in runs, whose sums are scanned.
template <int WARPS, typename Count>
__device__ __forceinline__ void scan_blocks(int n, Count count, int64_t* sums, int64_t& before,
                                            int64_t& mine, int64_t& total) {
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int run = (n + 32 * WARPS - 1) / (32 * WARPS);
  mine = 0;
  for (int i = tid * run; i < min((tid + 1) * run, n); ++i) mine += count(i);
  before = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t x = __shfl_up_sync(FULL_MASK, before, m);
    if (lane >= m) before += x;
  }
  if (lane == 31) sums[w] = before;
  __syncthreads();
  total = 0;
  before -= mine;
#pragma unroll
  for (int x = 0; x < WARPS; ++x) {
    if (x < w) before += sums[x];
    total += sums[x];
  }
}

// The sequence of this thread's run that holds block b, and the block's number
// in it; b lies in [before, before + mine).
template <int WARPS, typename Count>
__device__ __forceinline__ int find_block(int n, Count count, int64_t before, int64_t b,
                                          int64_t& in) {
  int i = threadIdx.x * ((n + 32 * WARPS - 1) / (32 * WARPS));
  for (int64_t nb = count(i); b >= before + nb; nb = count(++i)) before += nb;
  in = b - before;
  return i;
}

// ------------------------------------------------------------ write and read

constexpr int TW = 4;  // warps per CTA

// Codes of four values: x / scale lands in the low mantissa bits of 1.5 * 2^23 +
// 128, rounded once, to nearest even (the product alone is exact).
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  constexpr float MAGIC = 12582912.0f + 128.0f;
  const uint32_t x = __float_as_uint(fmaf(a, inv, MAGIC)), y = __float_as_uint(fmaf(b, inv, MAGIC));
  const uint32_t z = __float_as_uint(fmaf(c, inv, MAGIC)), w = __float_as_uint(fmaf(d, inv, MAGIC));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}
__device__ __forceinline__ float value_of(uint32_t word, int byte, float scale) {
  // byte u under 0x4b000000 is 2^23 + u
  const uint32_t u = __byte_perm(word, 0x4b000000u, 0x7440 + byte);
  return (__uint_as_float(u) - 8388736.0f) * scale;
}
// Older codes under a grown scale (ratio = old / new, a power of two below 1).
__device__ __forceinline__ uint32_t recode4(uint32_t word, float ratio) {
  return codes4(value_of(word, 0, 1.0f), value_of(word, 1, 1.0f), value_of(word, 2, 1.0f),
                value_of(word, 3, 1.0f), ratio);
}
__device__ __forceinline__ uint32_t absmax2(uint32_t m, uint32_t pair) {
  return __vmaxu2(m, pair & 0x7fff7fffu);  // bf16 magnitudes order as their bits
}
// NaN to 0, magnitudes beyond 127 * 2^120 to that, both halves of a word.
constexpr uint32_t MOST_BITS = 0x7efe;
__device__ __forceinline__ uint32_t storable2(uint32_t pair) {
  const uint32_t mag = pair & 0x7fff7fffu;
  return (__vminu2(mag, MOST_BITS * 0x10001u) | (pair & 0x80008000u)) & ~__vcmpgtu2(mag, 0x7f807f80u);
}

// A tile is the K or the V of one block and head, 16 tokens x D, held by D / 8
// lanes: lane ll has dims 8 ll .. 8 ll + 7 of every token, a 16-byte load or
// store per token, all in flight at once.  Rows and codes meet in 16 D bytes of
// shared memory per tile, which stand in the pool's order (16-byte chunks, D / 32
// groups of 32) with each group's chunks swapped about by its number, so that
// neither side's accesses share banks.  Bound by memory: 65536 tokens of 8 heads of
// 128 (403 MB) written in 70 us, 5.75 TB/s, 0.88 of the measured copy rate, read in
// 65 us, 0.95.  The first form, a thread per 16 bytes of the pool with 2-byte loads
// of V, took 222 us each.  A write holds its 16 rows in registers, which leaves 16
// warps per SM; 20 of them spilled (164 us for both instead of 151 then).
template <int D, bool WRITE>
__global__ void __launch_bounds__(32 * TW, WRITE ? 4 : 1) kv8_rows_kernel(const Kv8RowsArgs a) {
  constexpr int LPT = D / 8, TILES = 32 / LPT;  // lanes per tile, tiles per warp
  __shared__ __align__(128) uint8_t stage[TW][TILES * BT * D];
  __shared__ uint4 older[WRITE ? TW : 1][256];  // a partly new block's chunks before, each lane's own
  __shared__ int64_t sums[TW];
  __shared__ struct { int64_t nth; int32_t seq, pos, row, cnt; } at[TW / 2 * TILES];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int ll = lane % LPT, tile = lane / LPT;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Two warps take the K and the V of the same TILES (block, head) pairs, which
  // count the heads of a block, then the blocks.
  constexpr int PAIRS = TW / 2 * TILES;  // of a CTA
  const int sel = w & 1, slot = (w >> 1) * TILES + tile;
  const uint32_t heads = a.kv_heads, u0 = blockIdx.x * PAIRS, u = u0 + slot, ub = u / heads;
  const int head = int(u - ub * heads);
  int seq;
  int64_t nth = 0;  // of the sequence's touched blocks
  int64_t first = 0, row0 = 0, cnt = 1;  // its first position, row and number of rows
  if (a.start && a.n <= 128) {
    // every warp looks for itself, 32 sequences at a time, without a barrier
    const uint32_t most = gridDim.x * PAIRS;  // blocks of a sequence beyond that are out of any CTA's reach
    uint32_t before = 0;
    seq = -1;
    for (int i0 = 0; i0 < a.n; i0 += 32) {
      const int i = min(i0 + lane, a.n - 1);
      const int32_t p = a.pos[i], r = a.start[i];
      const int64_t c = i0 + lane < a.n ? int64_t(a.start[i + 1]) - r : 0;
      if (c > 0 && p < 0) record_error(&g_kv8_error, QC_ERR_BOUNDS);
      const uint32_t nb = p < 0 ? 0 : uint32_t(min(blocks_touched(p, c), int64_t(most)));
      uint32_t upto = nb;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const uint32_t x = __shfl_up_sync(FULL_MASK, upto, m);
        if (lane >= m) upto += x;
      }
      upto = min(upto, most);  // at most 32 * 2^26 before, however the rows overlap
#pragma unroll
      for (int x = 0; x < TILES; ++x) {
        const uint32_t b = __shfl_sync(FULL_MASK, ub, x * LPT);
        const int in = __popc(__ballot_sync(FULL_MASK, before + upto <= b));  // sequences that end before b
        const int from = min(in, 31);
        const int64_t c1 = __shfl_sync(FULL_MASK, c, from);
        const int32_t p1 = __shfl_sync(FULL_MASK, p, from), r1 = __shfl_sync(FULL_MASK, r, from);
        const uint32_t past = __shfl_sync(FULL_MASK, upto - nb, from);
        if (tile == x && seq < 0 && in < 32 && b >= before) {
          seq = i0 + in;
          nth = b - before - past;
          first = p1;
          row0 = r1;
          cnt = c1;
        }
      }
      before += __shfl_sync(FULL_MASK, upto, 31);
    }
    if (seq >= a.n) seq = -1;
    if (blockIdx.x == 0 && tid == 0 && uint64_t(before) * heads > uint64_t(gridDim.x) * PAIRS)
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
  } else if (a.start) {
    const auto count = [&](int i) -> int64_t {
      const int64_t cnt = int64_t(a.start[i + 1]) - a.start[i];
      if (cnt > 0 && a.pos[i] < 0) record_error(&g_kv8_error, QC_ERR_BOUNDS);
      return a.pos[i] < 0 ? 0 : blocks_touched(a.pos[i], cnt);
    };
    if (tid < PAIRS) at[tid].seq = -1;
    int64_t before, mine, total;
    scan_blocks<TW>(a.n, count, sums, before, mine, total);
    if (mine > 0) {
      uint32_t b = u0 / heads, left = (b + 1) * heads - u0;
      for (int x = 0; x < PAIRS; ++x) {
        if (b >= before && b < before + mine) {
          int64_t nth;
          const int i = find_block<TW>(a.n, count, before, b, nth);
          at[x] = {nth, i, a.pos[i], a.start[i], int32_t(min(int64_t(a.start[i + 1]) - a.start[i], int64_t(INT32_MAX)))};
        }
        if (--left == 0) {
          ++b;
          left = heads;
        }
      }
    }
    // rows that overlap or leave the input can ask for more blocks than the launch has
    if (blockIdx.x == 0 && tid == 0 && total * a.kv_heads > int64_t(gridDim.x) * PAIRS)
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
    __syncthreads();
    seq = at[slot].seq;
    nth = at[slot].nth;
    first = at[slot].pos;
    row0 = at[slot].row;
    cnt = at[slot].cnt;
  } else {
    seq = ub < uint32_t(a.n) ? int(ub) : -1;
    row0 = seq;
    if (seq >= 0) first = a.pos[seq];
    if (first < 0) {
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
      seq = -1;
    }
  }

  int lo = 0, hi = 0;  // the block's tokens that are rows of this call: [lo, hi)
  int64_t row = 0;     // input row of token 0
  uint8_t* block = nullptr;
  if (seq >= 0) {
    const int64_t begin = (first / BT + nth) * BT;
    lo = first > begin ? int(first - begin) : 0;
    hi = int(min(first + cnt - begin, int64_t(BT)));
    row = row0 + begin - first;
    const int64_t pg = begin / QC_PAGE;
    const int32_t page = pg < a.pt_stride ? a.table[int64_t(seq) * a.pt_stride + pg] : -1;
    if (page < 0 || page >= a.n_pages || row + lo < 0 || row + hi > a.rows) {
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
      hi = lo = 0;
    } else {
      block = a.pool + ((int64_t(page) * a.kv_heads + head) * PAGE_BLOCKS + begin % QC_PAGE / BT) *
                           block_bytes(D);
    }
  }
  const int64_t ld = sel ? a.v_ld : a.k_ld;
  uint16_t* rows = (sel ? a.v : a.k) + row * ld + head * D + 8 * ll;
  float* scale_at = reinterpret_cast<float*>(block) + sel;
  uint4* chunks = reinterpret_cast<uint4*>(block + HEAD_BYTES + sel * BT * D);
  uint8_t* mine = stage[w] + tile * BT * D;
  // Chunk idx = 4 g + t of group i stands at idx ^ key(i).
  const auto key = [&](int i) { return (tile * (LPT / 4) + i) & 7; };
  const auto chunk_at = [&](int i, int idx) { return mine + 512 * i + 16 * (idx ^ key(i)); };
  // Words of lane ll in that order: K, 4 dims of tokens rho(g) and rho(g) + 2 side by
  // side, for its runs of dims 8 ll .. + 3 and 8 ll + 4 .. + 7; V, 4 tokens of dim 8 ll + g.
  const int gi = ll / 4;
  const auto k_word = [&](int g, int e) {
    return reinterpret_cast<uint2*>(chunk_at(gi, 4 * g + ((2 * ll + e) & 3)) + 8 * ((ll & 3) >> 1));
  };
  const auto v_word = [&](int g, int t) {
    return reinterpret_cast<uint32_t*>(chunk_at(gi, 4 * g + t) + 4 * (ll & 3));
  };

  if (WRITE) {
    uint4 x[BT];
#pragma unroll
    for (int s = 0; s < BT; ++s)
      x[s] = s >= lo && s < hi ? *reinterpret_cast<const uint4*>(rows + s * ld) : make_uint4(0, 0, 0, 0);
    const bool part = hi > lo && (lo > 0 || hi < BT);
    float old_scale = 0.0f;
    if (part) {
      old_scale = *scale_at;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         smem_u32(&older[w][c * 32 + lane])),
                     "l"(chunks + c * LPT + ll)
                     : "memory");
    }
    const auto tile_max = [&]() {
      uint32_t m = 0;
#pragma unroll
      for (int s = 0; s < BT; ++s)
        m = absmax2(absmax2(absmax2(absmax2(m, x[s].x), x[s].y), x[s].z), x[s].w);
      m = max(m & 0xffffu, m >> 16);
      for (int d = LPT / 2; d; d >>= 1) m = max(m, __shfl_xor_sync(FULL_MASK, m, d));
      return m;
    };
    uint32_t top = tile_max();
    if (__any_sync(FULL_MASK, top > MOST_BITS)) {
#pragma unroll
      for (int s = 0; s < BT; ++s)
        x[s] = make_uint4(storable2(x[s].x), storable2(x[s].y), storable2(x[s].z), storable2(x[s].w));
      top = tile_max();
    }
    float scale = pow2_scale(__uint_as_float(top << 16));
    if (lo > 0) scale = fmaxf(scale, old_scale);  // older tokens stay: the scale does not shrink
    const float inv = 1.0f / scale, ratio = old_scale / scale;
    if (sel == 0) {
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const int rho = 4 * (g >> 1) + (g & 1);
        const uint4 p = x[rho], q = x[rho + 2];
        *k_word(g, 0) = make_uint2(codes4(bf_lo(p.x), bf_hi(p.x), bf_lo(p.y), bf_hi(p.y), inv),
                                   codes4(bf_lo(q.x), bf_hi(q.x), bf_lo(q.y), bf_hi(q.y), inv));
        *k_word(g, 1) = make_uint2(codes4(bf_lo(p.z), bf_hi(p.z), bf_lo(p.w), bf_hi(p.w), inv),
                                   codes4(bf_lo(q.z), bf_hi(q.z), bf_lo(q.w), bf_hi(q.w), inv));
      }
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint4 p = x[4 * t], q = x[4 * t + 1], r = x[4 * t + 2], z = x[4 * t + 3];
        *v_word(0, t) = codes4(bf_lo(p.x), bf_lo(q.x), bf_lo(r.x), bf_lo(z.x), inv);
        *v_word(1, t) = codes4(bf_hi(p.x), bf_hi(q.x), bf_hi(r.x), bf_hi(z.x), inv);
        *v_word(2, t) = codes4(bf_lo(p.y), bf_lo(q.y), bf_lo(r.y), bf_lo(z.y), inv);
        *v_word(3, t) = codes4(bf_hi(p.y), bf_hi(q.y), bf_hi(r.y), bf_hi(z.y), inv);
        *v_word(4, t) = codes4(bf_lo(p.z), bf_lo(q.z), bf_lo(r.z), bf_lo(z.z), inv);
        *v_word(5, t) = codes4(bf_hi(p.z), bf_hi(q.z), bf_hi(r.z), bf_hi(z.z), inv);
        *v_word(6, t) = codes4(bf_lo(p.w), bf_lo(q.w), bf_lo(r.w), bf_lo(z.w), inv);
        *v_word(7, t) = codes4(bf_hi(p.w), bf_hi(q.w), bf_hi(r.w), bf_hi(z.w), inv);
      }
    }
    __syncwarp();
    if (hi > lo && ll == 0) *scale_at = scale;
    if (hi > lo && !part) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        chunks[c * LPT + ll] =
            *reinterpret_cast<const uint4*>(chunk_at((c * LPT + ll) >> 5, (c * LPT + ll) & 31));
    } else if (hi > lo) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      // bytes of tokens below lo keep their value, those from hi on their bits;
      // a word is 4 tokens from 4 t (V) or one token (K: in turn rho(g) and rho(g) + 2)
      const auto below = [](int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; };
      uint32_t kept[2] = {below(lo - 4 * (ll & 3)), 0}, fresh[2] = {below(hi - 4 * (ll & 3)) & ~kept[0], 0};
      kept[1] = kept[0];
      fresh[1] = fresh[0];
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        const int i = (c * LPT + ll) >> 5, idx = (c * LPT + ll) & 31, g = idx >> 2;
        if (sel == 0)
          for (int e = 0; e < 2; ++e) {
            const int token = 4 * (g >> 1) + (g & 1) + 2 * e;
            kept[e] = token < lo ? ~0u : 0u;
            fresh[e] = token < hi ? ~kept[e] : 0u;
          }
        const uint4 y = *reinterpret_cast<const uint4*>(chunk_at(i, idx)), old = older[w][c * 32 + lane];
        const auto merge = [&](uint32_t n, uint32_t was, int e) {
          if (kept[e] && ratio != 1.0f) was = (recode4(was, ratio) & kept[e]) | (was & ~kept[e]);
          return (n & fresh[e]) | (was & ~fresh[e]);
        };
        chunks[c * LPT + ll] = make_uint4(merge(y.x, old.x, 0), merge(y.y, old.y, 1),
                                          merge(y.z, old.z, 0), merge(y.w, old.w, 1));
      }
    }
  } else {
    float scale = 0.0f;
    if (hi > lo) {
      scale = *scale_at;
      uint4 y[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) y[c] = chunks[c * LPT + ll];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<uint4*>(chunk_at((c * LPT + ll) >> 5, (c * LPT + ll) & 31)) = y[c];
    }
    __syncwarp();
    const auto pair = [&](uint32_t a0, int b0, uint32_t a1, int b1) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(value_of(a0, b0, scale), value_of(a1, b1, scale));
      return *reinterpret_cast<const uint32_t*>(&h);
    };
    const auto put = [&](int s, uint4 y) {
      if (s >= lo && s < hi) *reinterpret_cast<uint4*>(rows + s * ld) = y;
    };
    if (sel == 0) {
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const int rho = 4 * (g >> 1) + (g & 1);
        const uint2 p = *k_word(g, 0), q = *k_word(g, 1);
        put(rho, make_uint4(pair(p.x, 0, p.x, 1), pair(p.x, 2, p.x, 3), pair(q.x, 0, q.x, 1), pair(q.x, 2, q.x, 3)));
        put(rho + 2, make_uint4(pair(p.y, 0, p.y, 1), pair(p.y, 2, p.y, 3), pair(q.y, 0, q.y, 1), pair(q.y, 2, q.y, 3)));
      }
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t v[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) v[g] = *v_word(g, t);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          put(4 * t + e, make_uint4(pair(v[0], e, v[1], e), pair(v[2], e, v[3], e), pair(v[4], e, v[5], e),
                                    pair(v[6], e, v[7], e)));
      }
    }
  }
}

// ---------------------------------------------------------------- attention
//
// out = sum_j 2^(x_j - m) V_j / sum_j 2^(x_j - m), x_j = scale * log2(e) q.K_j,
// one pass over the blocks with a running maximum.
//
// Split.  A step is 8 KB of codes: one block of 256-wide heads, two of 128, four of
// 64, one bulk copy (a block is scales, K, V).  The steps of all (sequence, kv head)
// pairs, counted in order, are cut into one equal contiguous range per warp of the
// grid.  A warp streams its steps through its own ring and works on each alone.  A
// pair that lies whole in one range is finished there; of the others every range
// writes a record (m, l, r, o), which the merge kernel adds in order.  Where all
// ranges of a CTA lie in one pair its warps meet once, at the end, and write one
// record for the four.
//
// Products.  S = K q on m16n8k16 f16 with f32 sums: the codes are whole numbers
// up to 127 and the bf16 queries, scaled by a power of two, are exact in f16 down to
// 2^-30 of their head's largest (below that they round, by at most 2^-38 of it), so
// the products are exact.  Two byte permutes and two subtractions turn four
// codes into f16: byte u under 0x64 is 1024 + u, less 1152 the code.  The row
// order of the cache makes S, transposed by movmatrix, the operand of
// O^T = V^T w without any other exchange.
//
// The weights of the second product carry V's scale: w = 2^(x + log2 sv - r)
// with a running reference r of its own, so blocks of very different scales
// keep their precision (l has no part in it).  w stands in f16, at most 2^15, and
// w - f16(w) beside it, so that 22 bits of it count (of a w below 2^-3, which is 2^-10
// of the largest or less, those above 2^-25): in the product's other 4
// columns for groups of up to 4 heads, in a second product for larger ones (64 x
// 4096 with 6 heads of 128 to a KV head 86.5 -> 87.8 us, 33 sequences of up to 8191
// 20.0 -> 21.0).  Both references move only when a score passes them by 2^8 (m; r
// starts 2^7 under its largest and moves at 2^15), so most blocks rescale nothing.
//
// Bound by memory: 64 sequences of 4096 with 4 heads of 256 (538 MB) 87 us, 6.2 TB/s,
// 0.95 of the measured copy rate, the merge included.  A block costs a warp 32
// products of 8 cycles (48 for groups above 4) and some 590 other instructions, half of
// what the SM could issue meanwhile.  mma.sync and not tcgen05: with 1 to 8 query rows the tensor pipe
// has little to do, and the codes pass through registers on the way to f16 anyway.

struct Kv8AttnArgs {
  const uint8_t* pool;
  const int32_t *table, *len;
  const uint16_t *q, *gate;
  uint16_t* out;
  int4* owner;      // a split pair: its number; 8 * joined CTAs + records before them; records;
                    // slot of the first.  One entry per pair (by_pair) or for the last pair that
                    // each warp starts
  float* rec;       // [warps][2][group][D + 4]: m, l, r, unused, o
  int64_t q_ld, q_head, out_ld;
  float scale;      // scale * log2(e) = scale * 2^scale_exp, scale in [0.5, 1)
  int32_t scale_exp;
  int32_t n_pages, pt_stride, kv_heads, group, n;
  int32_t by_pair, warps;
};

constexpr int AW = 4;                                    // warps per CTA
// Blocks of a step, what a warp copies and works on at once (8 KB of codes, and
// the step's fixed part paid once); steps in flight per warp; CTAs per SM.  16
// copies of 8 KB in flight per SM are enough and more do harm: the SMs then share
// the bandwidth unevenly and the equal ranges end far apart.  D 256, 64 x 4096 and 1
// x 131072 (us): 8 warps of 2 steps 88.8 and 50.6, of 3 steps 96.9 and 56.3; 10 of 2
// 97.8 and 56.3; 6 of 2 95.6 and 53.2; 4 of 4 105 and 57.  D 128, 32 x 4096: 8 of 2
// 49.3, of 3 52.1; steps of one block 57.3.  D 64, 64 x 8000: 12 of 2 50.9, 10 of 2
// 55.6, 8 of 2 65.8 (more arithmetic per byte).
__host__ __device__ constexpr int step_blocks(int dim) { return 256 / dim; }
__host__ __device__ constexpr int stages(int dim) { return 2; }
__host__ __device__ constexpr int ctas_per_sm(int dim) { return dim == 64 ? 3 : 2; }
constexpr int MAX_WARPS = 1824;                          // of the grid
constexpr float LAZY_M = 8.0f, TOP_R = 7.0f, LAZY_R = 15.0f;

template <int D>
struct AttnSmem {
  static constexpr int AS = stages(D);
  alignas(128) uint8_t stage[AW][AS][step_blocks(D) * block_bytes(D)];
  alignas(8) uint64_t full[AW][AS];
  int32_t valid[AW][AS];                                 // tokens of the step; 0: nothing was copied
  int64_t sums[AW];
  float m[AW][8], l[AW][8], r[AW][8];  // of a joined CTA's warps
  struct { int64_t unit; int32_t seq, n, len; } start[AW];
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// l under a reference that moved from m to m1; 0 exactly where no token was met, NaN passes.
__device__ __forceinline__ float rebase(float l, float m, float m1) {
  return l == 0.0f || m == m1 ? l : l * ex2(m - m1);
}
// o 2^(r - m) / l as two factors, the power in two halves: either alone may leave f32.
__device__ __forceinline__ float2 finish(float m, float l, float r) {
  const float half = 0.5f * (r - m);
  return l == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(ex2(half) / l, ex2(r - m - half));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes 0, 1 (and 2, 3) of a word as f16 pairs.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  const uint32_t u = __byte_perm(w, 0x64646464u, 0x4140);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  const uint32_t u = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// bulk_g2s of bytes that are read once: they leave L2 before what is there already
// (64 x 4096, three caches in turn: 91.8 -> 88.0 us).
__device__ __forceinline__ uint64_t streaming_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void bulk_g2s_stream(void* dst, const void* src, uint32_t bytes,
                                                uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// Tokens of a sequence, as many as its page-table row can name, and their steps.
__device__ __forceinline__ int32_t seq_len(const Kv8AttnArgs& a, int32_t i) {
  return int32_t(min(int64_t(max(a.len[i], 0)), int64_t(a.pt_stride) * QC_PAGE));
}
template <int D>
__device__ __forceinline__ int64_t seq_steps(const Kv8AttnArgs& a, int32_t i) {
  constexpr int ST = BT * step_blocks(D);
  return (int64_t(seq_len(a, i)) + ST - 1) / ST;
}

// Where in the order of steps a warp stands: `unit` counts the steps of all
// pairs, `at` those of the pair (seq, head), which has n.
template <int D>
struct Cursor {
  int64_t unit;
  int32_t seq, head, at, n, len;

  __device__ __forceinline__ void enter(const Kv8AttnArgs& a) {
    n = int32_t(seq_steps<D>(a, seq));
    len = seq_len(a, seq);
  }
  // To the next pair that has tokens; the caller knows that there is one.
  __device__ __forceinline__ void next_pair(const Kv8AttnArgs& a) {
    at = 0;
    if (++head == a.kv_heads) {
      head = 0;
      do {
        ++seq;
      } while (seq + 1 < a.n && seq_len(a, seq) == 0);
      enter(a);
    }
  }
};

// Sequences without tokens: a row of zeros and nothing to merge.  Lengths out of
// range are reported.  Dealt to the warps of the grid.
template <int D>
__device__ __forceinline__ void mark_empty(const Kv8AttnArgs& a) {
  const int lane = threadIdx.x & 31;
  for (int i = (threadIdx.x >> 5) * gridDim.x + blockIdx.x; i < a.n; i += gridDim.x * AW) {
    const int32_t len = a.len[i];
    if (lane == 0 && (len < 0 || len > int64_t(a.pt_stride) * QC_PAGE))
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
    if (len > 0) continue;
    for (int d = lane * 8; d < a.kv_heads * a.group * D; d += 8 * 32)
      *reinterpret_cast<uint4*>(a.out + i * a.out_ld + d) = make_uint4(0, 0, 0, 0);
    for (int h = lane; h < a.kv_heads && a.by_pair; h += 32)
      a.owner[i * a.kv_heads + h] = make_int4(0, 0, 0, 0);
  }
}

template <int D, bool PAIRED>
__global__ void __launch_bounds__(32 * AW, ctas_per_sm(D)) kv8_attn_kernel(const Kv8AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  AttnSmem<D>& sm = *reinterpret_cast<AttnSmem<D>*>(smem_raw);
  constexpr int KS = D / 16;  // steps of 16 dims
  constexpr int AS = stages(D), GB = step_blocks(D), ST = BT * GB;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < AS; ++s) mbar_init(&sm.full[w][s], 1);
    fence_mbar_init();
  }
  __syncwarp();  // a warp's barriers are its own
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int warps = gridDim.x * AW;
  int64_t total, per;
  bool spread;
  const auto share = [&]() {
    per = max(quotient(total + warps - 1, warps), int64_t(1));
    // ranges side by side are one CTA's, so that it can join them; when there is at most
    // one step for each warp and few for a pair they go to different SMs: 4 heads of 256, 64
    // steps each, 8.5 us so and 9.3 joined, 128 steps 9.2 and 9.5, 160 the same, 200 10.0 and
    // 9.6 (one head alone turns at some 40 steps, 0.2 to 0.8 us apart up to 128)
    spread = total <= warps && total <= int64_t(128) * a.n * a.kv_heads;
  };
  const auto range_of = [&](int x) { return spread ? x * int(gridDim.x) + int(blockIdx.x) : int(blockIdx.x) * AW + x; };
  struct { int64_t unit; int32_t seq, n, len; } start;  // the sequence this warp starts in, its first unit
  if (a.n <= 32) {  // a sequence per lane, every warp for itself
    const int32_t len = seq_len(a, min(lane, a.n - 1));
    const int32_t steps = lane < a.n ? int32_t((int64_t(len) + ST - 1) / ST) : 0;
    int64_t upto = steps;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int64_t x = __shfl_up_sync(FULL_MASK, upto, m);
      if (lane >= m) upto += x;
    }
    total = __shfl_sync(FULL_MASK, upto, 31) * a.kv_heads;
    share();
    const int in = min(__popc(__ballot_sync(FULL_MASK, upto * a.kv_heads <= range_of(w) * per)), 31);
    start.unit = __shfl_sync(FULL_MASK, upto - steps, in) * a.kv_heads;
    start.seq = in;
    start.n = __shfl_sync(FULL_MASK, steps, in);
    start.len = __shfl_sync(FULL_MASK, len, in);
  } else {
    const auto count = [&](int i) { return seq_steps<D>(a, i); };
    int64_t before, mine;
    scan_blocks<AW>(a.n, count, sm.sums, before, mine, total);
    total *= a.kv_heads;
    share();
    for (int x = 0; x < AW; ++x) {
      const int64_t u = range_of(x) * per;  // warp x's first step
      if (u >= before * a.kv_heads && u < (before + mine) * a.kv_heads) {
        int64_t at = before;
        int i = tid * ((a.n + 32 * AW - 1) / (32 * AW));
        int64_t nb = count(i);
        for (; u >= (at + nb) * a.kv_heads; nb = count(++i)) at += nb;
        sm.start[x] = {at * a.kv_heads, i, int32_t(nb), seq_len(a, i)};
      }
    }
    __syncthreads();
    start.unit = sm.start[w].unit;
    start.seq = sm.start[w].seq;
    start.n = sm.start[w].n;
    start.len = sm.start[w].len;
  }
  const int wid = range_of(w);
  const int64_t begin = wid * per, end = min(begin + per, total);
  if (lane == 0 && !a.by_pair) a.owner[wid] = make_int4(0, 0, 0, 0);
  if (begin >= end) {
    mark_empty<D>(a);
    return;
  }

  Cursor<D> c;
  c.unit = begin;
  c.seq = start.seq;
  c.n = start.n;
  c.len = start.len;
  c.head = int32_t(quotient(begin - start.unit, c.n));
  c.at = int32_t(begin - start.unit - int64_t(c.head) * c.n);
  // whether the CTA's ranges, none of them empty, lie in one pair: the same for its warps
  const int64_t u0 = int64_t(blockIdx.x) * AW * per, pair0 = begin - c.at;
  const bool joined = !spread && u0 >= pair0 && min(u0 + AW * per, total) <= pair0 + c.n && u0 + (AW - 1) * per < total;
  Cursor<D> p = c;  // the copies run AS steps ahead
  int put = 0;
  const uint64_t policy = streaming_policy();
  auto issue = [&]() {  // lane 0: the copy of step p into the next stage
    if (p.unit >= end) return;
    const int32_t block = p.at * GB;
    // not by a read-only load: this kernel may be up while the table is still being written
    const int32_t page = a.table[int64_t(p.seq) * a.pt_stride + block / PAGE_BLOCKS];
    const bool ok = page >= 0 && page < a.n_pages;
    const int32_t tokens = min(p.len - block * BT, GB * BT);
    sm.valid[w][put] = ok ? tokens : 0;
    if (ok) {
      const uint32_t bytes = (tokens + BT - 1) / BT * block_bytes(D);
      mbar_arrive_expect_tx(&sm.full[w][put], bytes);
      bulk_g2s_stream(
          sm.stage[w][put],
          a.pool + ((int64_t(page) * a.kv_heads + p.head) * PAGE_BLOCKS + block % PAGE_BLOCKS) *
                       block_bytes(D),
          bytes, &sm.full[w][put], policy);
    } else {
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
      mbar_arrive(&sm.full[w][put]);
    }
    put = put + 1 == AS ? 0 : put + 1;
    ++p.unit;
    if (++p.at == p.n && p.unit < end) p.next_pair(a);
  };
  // A pair's queries are loaded before the copies are issued (behind megabytes of
  // them they would come late), a later pair's while the one before is stored.
  uint2 raw[KS];
  const auto load_q = [&]() {
    const int h = PAIRED ? g & 3 : g;
    const uint16_t* q = a.q + c.seq * a.q_ld + (int64_t(c.head) * a.group + h) * a.q_head + 4 * t;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      raw[s] = make_uint2(0, 0);
      if (h < a.group) raw[s] = *reinterpret_cast<const uint2*>(q + 16 * s);
    }
  };
  load_q();
  if (lane == 0)
    for (int s = 0; s < AS; ++s) issue();
  mark_empty<D>(a);

  int get = 0;
  uint32_t parity = 0;
  bool first = true, dead = false;
  while (c.unit < end && !dead) {
    // ---- the pair's queries, as operand columns: column n is head n (PAIRED: n % 4)
    const int32_t from = c.at;
    uint32_t qf[KS][2];
    float qs[2], qt[2];  // a column's products count for qs * qt
    {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) top = absmax2(absmax2(top, raw[s].x), raw[s].y);
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(FULL_MASK, top, 1));
      top = max(top, __shfl_xor_sync(FULL_MASK, top, 2));
      // q / 2^e: the largest value into [2^13, 2^14), so that values down to 2^-30 of it stay
      // exact: their 8 bits end at 2^-24, as f16 does.
      // The products count for scale * 2^at, one factor of which is applied before K's scale
      // and one after it, so that a score whose factors are far apart (q near 2^120, K near
      // 2^-120) leaves f32 at no step.
      const int e = max(int(top >> 7) - 127 - 13, -126), at = e + a.scale_exp;
      const int late = at > 0 ? at / 2 : at < -100 ? -64 : 0;
      const float up = __uint_as_float(uint32_t(127 - e) << 23);
      const float after = __uint_as_float(uint32_t(127 + late) << 23);
      float back = a.scale * __uint_as_float(uint32_t(max(127 + at - late, 1)) << 23);
      if (top >= 0x7f80u) back = __uint_as_float(0x7fc00000u);  // the whole row is NaN
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bool odd = top >= 0x7f80u;
        qf[s][0] = odd ? 0u : pack_f16(bf_lo(raw[s].x) * up, bf_hi(raw[s].x) * up);
        qf[s][1] = odd ? 0u : pack_f16(bf_lo(raw[s].y) * up, bf_hi(raw[s].y) * up);
      }
      qs[0] = __shfl_sync(FULL_MASK, back, 8 * t);
      qs[1] = __shfl_sync(FULL_MASK, back, 8 * t + 4);
      qt[0] = __shfl_sync(FULL_MASK, after, 8 * t);
      qt[1] = __shfl_sync(FULL_MASK, after, 8 * t + 4);
    }
    float m[2] = {-INFINITY, -INFINITY}, r[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[KS][4];
#pragma unroll
    for (int s = 0; s < KS; ++s) o[s][0] = o[s][1] = o[s][2] = o[s][3] = 0.0f;

    const int32_t stop = int32_t(min(int64_t(c.n), c.at + (end - c.unit)));
    for (; c.at < stop; ++c.at, ++c.unit) {
      if (!__all_sync(FULL_MASK, mbar_wait(&sm.full[w][get], parity, &g_kv8_error))) {
        // leave nothing in flight: the other copies of this warp, each again bounded
        for (int s = 0; s < AS; ++s) {
          const int x = get + s < AS ? get + s : get + s - AS;
          if (c.unit + s < end) mbar_wait(&sm.full[w][x], get + s < AS ? parity : parity ^ 1, nullptr);
        }
        if (!joined) return;
        dead = true;  // the others of the CTA wait for this warp
        break;
      }
      const int valid = sm.valid[w][get];
      const uint8_t* step = sm.stage[w][get];
      // x[b][0], [1]: block b's token rho, columns 2t, 2t + 1; [2], [3]: token rho + 2
      const int rho = 4 * (g >> 1) + (g & 1);
      float x[GB][4], lsv[GB], top[2] = {-INFINITY, -INFINITY}, top_v[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int b = 0; b < GB; ++b) {
        x[b][0] = x[b][1] = x[b][2] = x[b][3] = -INFINITY;
        lsv[b] = 0.0f;
        if (b * BT < valid) {
          const uint8_t* block = step + b * block_bytes(D);
          const float2 sc = *reinterpret_cast<const float2*>(block);
          const uint4* kc = reinterpret_cast<const uint4*>(block + HEAD_BYTES) + lane;
          float acc[2][4] = {};
#pragma unroll
          for (int i = 0; i < KS / 2; ++i) {
            const uint4 y = kc[32 * i];
            mma_f16(acc[0], codes_lo(y.x), codes_lo(y.y), codes_hi(y.x), codes_hi(y.y), qf[2 * i][0],
                    qf[2 * i][1]);
            mma_f16(acc[1], codes_lo(y.z), codes_lo(y.w), codes_hi(y.z), codes_hi(y.w),
                    qf[2 * i + 1][0], qf[2 * i + 1][1]);
          }
          lsv[b] = float(int((__float_as_uint(sc.y) >> 23) & 0xffu) - 127);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[b][j] = (acc[0][j] + acc[1][j]) * qs[j & 1] * sc.x * qt[j & 1];
            if (b * BT + rho + (j & 2) >= valid) x[b][j] = -INFINITY;
            top[j & 1] = fmaxf(top[j & 1], x[b][j]);
            top_v[j & 1] = fmaxf(top_v[j & 1], x[b][j] + lsv[b]);
          }
        }
      }
      const bool move = top[0] > m[0] + LAZY_M || top[1] > m[1] + LAZY_M ||
                        top_v[0] > r[0] + LAZY_R || top_v[1] > r[1] + LAZY_R;
      if (__any_sync(FULL_MASK, move)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            top[j] = fmaxf(top[j], __shfl_xor_sync(FULL_MASK, top[j], d));
            top_v[j] = fmaxf(top_v[j], __shfl_xor_sync(FULL_MASK, top_v[j], d));
          }
          const float m1 = fmaxf(m[j], top[j]), r1 = fmaxf(r[j], top_v[j] - TOP_R);
          if (m1 > m[j]) {
            l[j] *= ex2(m[j] - m1);
            m[j] = m1;
          }
          if (r1 > r[j]) {
            const float f = ex2(r[j] - r1);
            r[j] = r1;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              o[s][j] *= f;
              o[s][j + 2] *= f;
            }
          }
        }
      }
#pragma unroll
      for (int b = 0; b < GB; ++b) {
        if (b * BT >= valid) break;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = b * BT + rho + (j & 2) < valid;
          l[j & 1] += in ? ex2(x[b][j] - m[j & 1]) : 0.0f;
          y[j] = in ? ex2(x[b][j] + lsv[b] - r[j & 1]) : 0.0f;
          if (PAIRED && t >= 2) y[j] -= __half2float(__float2half_rn(y[j]));
        }
        const uint32_t b0 = transpose8(pack_f16(y[0], y[1]));
        const uint32_t b1 = transpose8(pack_f16(y[2], y[3]));
        uint32_t r0 = 0, r1 = 0;  // the rest, where it has no columns of its own
        if (!PAIRED) {
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] -= __half2float(__float2half_rn(y[j]));
          r0 = transpose8(pack_f16(y[0], y[1]));
          r1 = transpose8(pack_f16(y[2], y[3]));
        }
        const uint4* vc =
            reinterpret_cast<const uint4*>(step + b * block_bytes(D) + HEAD_BYTES) + D + lane;
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
          const uint4 v = vc[32 * i];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x0 = half ? v.z : v.x, x1 = half ? v.w : v.y;
            const uint32_t a0 = codes_lo(x0), a1 = codes_lo(x1), a2 = codes_hi(x0), a3 = codes_hi(x1);
            mma_f16(o[2 * i + half], a0, a1, a2, a3, b0, b1);
            if (!PAIRED) mma_f16(o[2 * i + half], a0, a1, a2, a3, r0, r1);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0) issue();
      get = get + 1 == AS ? 0 : get + 1;
      if (get == 0) parity ^= 1;
    }

    // ---- the pair's result, or its record
    const int32_t seq = c.seq, kvh = c.head;
    const int64_t pair_end = c.unit - c.at + c.n;  // its last step's unit, plus one
    const bool done = c.at == c.n, whole = done && from == 0;
    if (done && c.unit < end) {
      c.next_pair(a);
      load_q();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[j] += __shfl_xor_sync(FULL_MASK, l[j], 4);
      l[j] += __shfl_xor_sync(FULL_MASK, l[j], 8);
      l[j] += __shfl_xor_sync(FULL_MASK, l[j], 16);
    }
    if (PAIRED) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[s][j] += __shfl_xor_sync(FULL_MASK, o[s][j], 2);
    }
    if (joined) {
      // every copy of the CTA has landed and been read by the time that its warps meet:
      // each leaves its sums in its own ring, [dim][two heads], and its references
      constexpr int HP = PAIRED ? 2 : 4;  // pairs of heads
      float2* mine = reinterpret_cast<float2*>(sm.stage[w]);
      __syncwarp();
      if (t < HP) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          mine[(16 * s + g) * HP + t] = make_float2(o[s][0], o[s][1]);
          mine[(16 * s + 8 + g) * HP + t] = make_float2(o[s][2], o[s][3]);
        }
        if (g == 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            sm.m[w][2 * t + j] = m[j];
            sm.l[w][2 * t + j] = l[j];
            sm.r[w][2 * t + j] = r[j];
          }
        }
      }
      __syncthreads();
      const int hp = tid % HP;
      float M[2], L[2], R[2], f[AW][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        M[j] = R[j] = -INFINITY;
        L[j] = 0.0f;
#pragma unroll
        for (int x = 0; x < AW; ++x) {
          M[j] = fmaxf(M[j], sm.m[x][2 * hp + j]);
          R[j] = fmaxf(R[j], sm.r[x][2 * hp + j]);
        }
#pragma unroll
        for (int x = 0; x < AW; ++x) {
          L[j] += rebase(sm.l[x][2 * hp + j], sm.m[x][2 * hp + j], M[j]);
          const float r1 = sm.r[x][2 * hp + j];
          f[x][j] = r1 == R[j] ? 1.0f : ex2(r1 - R[j]);
        }
      }
      float* rec = a.rec + (int64_t(blockIdx.x) * AW * 2 * a.group + 2 * hp) * (D + 4);
      const bool two = 2 * hp + 1 < a.group;
#pragma unroll
      for (int i = 0; i < D * HP / (32 * AW); ++i) {
        const int item = i * 32 * AW + tid, d = item / HP;
        float2 y = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int x = 0; x < AW; ++x) {
          const float2 z = reinterpret_cast<const float2*>(sm.stage[x])[item];
          y.x += z.x * f[x][0];
          y.y += z.y * f[x][1];
        }
        if (2 * hp < a.group) rec[4 + d] = y.x;
        if (two) rec[D + 8 + d] = y.y;
      }
      if (tid < HP) {
        if (2 * hp < a.group) *reinterpret_cast<float4*>(rec) = make_float4(M[0], L[0], R[0], 0.0f);
        if (two) *reinterpret_cast<float4*>(rec + D + 4) = make_float4(M[1], L[1], R[1], 0.0f);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (joined) break;
      // o[.][j]: dim g of the 16 and head 2t + j, o[.][j + 2]: dim g + 8.  PAIRED: both lanes
      // t and t + 2 have heads 2t, 2t + 1 by now; the first stores the dims g, the other g + 8
      const int h = PAIRED ? 2 * (t & 1) + j : 2 * t + j;
      constexpr int EACH = PAIRED ? 1 : 2;  // of the two
      const int d0 = PAIRED ? 8 * (t >> 1) + g : g;
      const auto value = [&](int s, int k) {
        return PAIRED ? (t < 2 ? o[s][j] : o[s][j + 2]) : o[s][j + 2 * k];
      };
      if (h >= a.group) continue;
      if (whole) {
        const float2 f = finish(m[j], l[j], r[j]);
        const int64_t head = int64_t(kvh) * a.group + h;
        uint16_t* out = a.out + seq * a.out_ld + head * D + d0;
        // the gate's logits all come before the first result is stored
        uint32_t gate[KS];  // of both dims
        if (a.gate) {
          const uint16_t* from = a.gate + seq * a.q_ld + head * a.q_head + d0;
#pragma unroll
          for (int s = 0; s < KS; ++s)
            gate[s] = from[16 * s] | (PAIRED ? 0u : uint32_t(from[16 * s + 8]) << 16);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < EACH; ++k) {
            float y = value(s, k) * f.x * f.y;
            if (a.gate) y *= sigmoid_exact(k ? bf_hi(gate[s]) : bf_lo(gate[s]));
            out[16 * s + 8 * k] = f2bf(y);
          }
      } else {
        float* rec = a.rec + ((int64_t(wid) * 2 + (first ? 0 : 1)) * a.group + h) * (D + 4);
        if (d0 == 0) *reinterpret_cast<float4*>(rec) = make_float4(m[j], l[j], r[j], 0.0f);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < EACH; ++k) rec[4 + d0 + 16 * s + 8 * k] = value(s, k);
      }
    }
    // the range that a pair starts in says what there is to merge
    if (lane == 0 && from == 0 && (!done || joined || a.by_pair)) {
      const int64_t number = int64_t(seq) * a.kv_heads + kvh;
      int4 own = make_int4(int(number), 0, 0, 2 * wid + (first ? 0 : 1));
      if (!whole || joined) {
        // its warps; the CTAs that it fills, from cta0 on; the records before them
        const int n = int(quotient(pair_end - 1, per)) - wid + 1;
        const int cta0 = (first ? wid + AW - 1 : wid + AW) / AW;
        const int64_t full = pair_end == total ? quotient(total + per - 1, per) / AW
                                               : quotient(pair_end, AW * per);
        const int ctas = spread ? 0 : int(max(full - cta0, int64_t(0))), before = ctas ? cta0 * AW - wid : 0;
        own.y = 8 * ctas + before;
        own.z = n - (AW - 1) * ctas;
      }
      a.owner[a.by_pair ? number : wid] = own;
    }
    first = false;
  }
}

// ---- merge of the records of split pairs
//
// A CTA takes an owner entry, 2^LOG_HG heads of the group and 2^LOG_CHUNK dims (all
// of them where it takes several heads): a lane for every 4 dims across, the rest
// of the 256 threads along the records, which are the owner's and then the first
// ones of the warps after it (of a joined CTA's its one).  Each thread's first records are loaded with the
// records' heads, from which the references and sums come; then the o are added in
// order.  It is latency throughout, so the launch keeps the CTAs to one wave
// (MERGE_CTAS): few heads have many records each and are spread over many CTAs, many
// heads share one.  16 x 4096: 256 CTAs 31.4 us in all, 2048 (32 dims each) 38.8, 4096
// (16 dims) 54.9; 1 x 131072: 256 CTAs of 16 dims 53.4, 128 of 32 dims 55.9.
constexpr int MERGE_CTAS = 592;

template <int D, int LOG_CHUNK, int LOG_HG>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Kv8AttnArgs a) {
  // a thread's records in flight with the heads; 2, 5 and 8 of them (us): 1 x 1024 9.2, 8.8,
  // 9.2; 16 x 4096 27.5, 27.3, 28.7; 1 x 131072 with one KV head of 256 20.3, 18.8, 19.0
  constexpr int AHEAD = 5;
  __shared__ float4 part[256];
  __shared__ float ref[LOG_HG == 0 ? MAX_WARPS : 1];  // one head: the records' r
  __shared__ float2 top_s[8];  // per warp: largest m and r of its head's records
  __shared__ float sum_s[8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int4 own = a.owner[blockIdx.x];
  const int n = own.z, ctas = own.y >> 3, before = own.y & 7, wid0 = own.w >> 1;
  // an entry whose warp gave up on a wait is whatever the workspace held: follow it
  // only inside the records and the batch
  if (n <= 0 || n > a.warps || own.y < 0 || ctas > n || before > AW || own.w < 0 ||
      wid0 > a.warps - n - (AW - 1) * ctas || own.x < 0 || own.x >= a.n * a.kv_heads)
    return;
  const int seq = own.x / a.kv_heads, kvh = own.x - seq * a.kv_heads;
  // record i: the owner's, then a warp's each, the joined CTAs', again a warp's each
  const auto record = [&](int i, int h) {
    const int skip = (AW - 1) * min(max(i - before, 0), ctas);
    return a.rec + (int64_t(i == 0 ? own.w : 2 * (wid0 + i + skip)) * a.group + h) * (D + 4);
  };
  constexpr int QUADS = (1 << LOG_CHUNK) / 4, LANES = QUADS << LOG_HG, SLOTS = 256 / LANES;
  const int quad = tid % LANES, slot = tid / LANES, hq = quad / QUADS;
  const int h = (blockIdx.y << LOG_HG) + hq, d = (blockIdx.z << LOG_CHUNK) + quad % QUADS * 4;
  const bool on = h < a.group;
  const int64_t head = int64_t(kvh) * a.group + h;
  uint2 gate = make_uint2(0, 0);
  if (a.gate && on && slot == 0)
    gate = *reinterpret_cast<const uint2*>(a.gate + seq * a.q_ld + head * a.q_head + d);
  float4 ahead[AHEAD];
  float at[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (on && slot + j * SLOTS < n) {
      const float* p = record(slot + j * SLOTS, h);
      if (LOG_HG > 0) at[j] = p[2];
      ahead[j] = *reinterpret_cast<const float4*>(p + 4 + d);
    }
  // the heads of the records: PER threads, whole warps, for each head
  constexpr int PER = 256 >> LOG_HG, NW = 8 >> LOG_HG;
  const int hs = (blockIdx.y << LOG_HG) + tid / PER;
  float m = -INFINITY, r = -INFINITY, l = 0.0f;
  const int heads_n = hs < a.group ? n : 0;
#pragma unroll 4
  for (int i = tid % PER; i < heads_n; i += PER) {
    const float4 s = *reinterpret_cast<const float4*>(record(i, hs));
    const float m1 = fmaxf(m, s.x);
    l = rebase(l, m, m1) + rebase(s.y, s.x, m1);
    m = m1;
    r = fmaxf(r, s.z);
    if (LOG_HG == 0) ref[i] = s.z;
  }
  const float mw = warp_max(m), rw = warp_max(r);
  if (lane == 0) top_s[w] = make_float2(mw, rw);
  __syncthreads();
  const auto top = [&](int first) {
    float2 t = top_s[first];
    for (int x = 1; x < NW; ++x) {
      t.x = fmaxf(t.x, top_s[first + x].x);
      t.y = fmaxf(t.y, top_s[first + x].y);
    }
    return t;
  };
  l = warp_sum(rebase(l, m, top(w / NW * NW).x));
  if (lane == 0) sum_s[w] = l;
  const float2 mr = top(hq * NW);
  float4 o = make_float4(0, 0, 0, 0);
  const auto add = [&](float r1, const float4& x) {
    const float f = r1 == mr.y ? 1.0f : ex2(r1 - mr.y);
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (on && slot + j * SLOTS < n) add(LOG_HG == 0 ? ref[slot + j * SLOTS] : at[j], ahead[j]);
  const int values_n = on ? n : 0;
#pragma unroll 4
  for (int i = slot + AHEAD * SLOTS; i < values_n; i += SLOTS) {
    const float* p = record(i, h);
    add(LOG_HG == 0 ? ref[i] : p[2], *reinterpret_cast<const float4*>(p + 4 + d));
  }
  // the slots of a warp, then those that are left (8 at most)
#pragma unroll
  for (int x = LANES; x < 32; x <<= 1) {
    o.x += __shfl_xor_sync(FULL_MASK, o.x, x);
    o.y += __shfl_xor_sync(FULL_MASK, o.y, x);
    o.z += __shfl_xor_sync(FULL_MASK, o.z, x);
    o.w += __shfl_xor_sync(FULL_MASK, o.w, x);
  }
  part[tid] = o;
  __syncthreads();
  if (slot != 0 || !on) return;
  float total = 0.0f;
  for (int x = 0; x < NW; ++x) total += sum_s[hq * NW + x];
  constexpr int NEXT = LANES > 32 ? LANES : 32;
#pragma unroll
  for (int s = NEXT; s < 256; s += NEXT) {
    const float4 x = part[s + quad];
    o.x += x.x;
    o.y += x.y;
    o.z += x.z;
    o.w += x.w;
  }
  const float2 f = finish(mr.x, total, mr.y);
  float y[4] = {o.x * f.x * f.y, o.y * f.x * f.y, o.z * f.x * f.y, o.w * f.x * f.y};
  if (a.gate) {
    y[0] *= sigmoid_exact(bf_lo(gate.x));
    y[1] *= sigmoid_exact(bf_hi(gate.x));
    y[2] *= sigmoid_exact(bf_lo(gate.y));
    y[3] *= sigmoid_exact(bf_hi(gate.y));
  }
  *reinterpret_cast<uint2*>(a.out + seq * a.out_ld + head * D + d) =
      make_uint2(f2bf(y[0]) | uint32_t(f2bf(y[1])) << 16, f2bf(y[2]) | uint32_t(f2bf(y[3])) << 16);
}

// Workspace: owners of MAX_WARPS warps, then their records.
int64_t owner_bytes() { return int64_t(MAX_WARPS) * sizeof(int4); }
int64_t record_bytes(int32_t group, int32_t dim) { return int64_t(group) * (dim + 4) * sizeof(float); }

template <int D, int LOG_CHUNK, int LOG_HG>
cudaError_t launch_merge_as(const Kv8AttnArgs& a, int entries, cudaStream_t s) {
  constexpr int HG = 1 << LOG_HG;
  const int64_t groups = (a.group + HG - 1) / HG;
  const bool fits = entries * groups * (D >> LOG_CHUNK) <= MERGE_CTAS;
  if constexpr ((1 << LOG_CHUNK) < D) {
    if (!fits) return launch_merge_as<D, LOG_CHUNK + 1, LOG_HG>(a, entries, s);
  } else if constexpr (HG < 8 && HG * D < 1024) {
    if (!fits && HG < a.group) return launch_merge_as<D, LOG_CHUNK, LOG_HG + 1>(a, entries, s);
  }
  return launch_dependent(kv8_merge_kernel<D, LOG_CHUNK, LOG_HG>,
                          dim3(entries, (unsigned)groups, D >> LOG_CHUNK), 256, 0, s, a);
}
template <int D>
cudaError_t launch_merge(const Kv8AttnArgs& a, int entries, cudaStream_t s) {
  return launch_merge_as<D, 4, 0>(a, entries, s);
}

template <int D, bool PAIRED>
cudaError_t launch_attn(Kv8AttnArgs a, cudaStream_t s) {
  static PerDeviceOnce configured;
  static std::atomic<int> ctas[64];  // CTAs that the device runs at once
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int grid = dev < 64 ? ctas[dev].load(std::memory_order_relaxed) : 0;
  if (!configured.done(dev) || grid == 0) {
    e = cudaFuncSetAttribute(kv8_attn_kernel<D, PAIRED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)sizeof(AttnSmem<D>));
    int sms = 0, per = 0;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kv8_attn_kernel<D, PAIRED>, 32 * AW,
                                                        sizeof(AttnSmem<D>));
    if (e != cudaSuccess) return e;
    grid = std::max(1, std::min(sms * std::min(per, ctas_per_sm(D)), MAX_WARPS / AW));
    if (dev < 64) ctas[dev].store(grid, std::memory_order_relaxed);
    configured.mark(dev);
  }
  const int warps = grid * AW;
  const int64_t pairs = int64_t(a.n) * a.kv_heads;
  a.by_pair = pairs <= warps;
  a.warps = warps;
  const int entries = a.by_pair ? int(pairs) : warps;
  e = launch_dependent(kv8_attn_kernel<D, PAIRED>, dim3(grid), 32 * AW, sizeof(AttnSmem<D>), s, a);
  if (e != cudaSuccess) return e;
  return launch_merge<D>(a, entries, s);
}

int check_cache(const char* call, const qc_kv8_cache* c) {
  if (!c) return refuse(QC_ERR_ARG, "%s: null cache", call);
  if (!qc_kv8_page_bytes(c->n_kv_heads, c->head_dim))
    return refuse(QC_ERR_ARG, "%s: %d KV heads of %d dims (1..%d heads of 64, 128 or 256)", call,
                  c->n_kv_heads, c->head_dim, QC_KV8_MAX_HEADS);
  if (c->n_pages < 1) return refuse(QC_ERR_ARG, "%s: n_pages %d", call, c->n_pages);
  if (!aligned16(c->pool)) return refuse(QC_ERR_ARG, "%s: the pool is not 16-byte aligned", call);
  return QC_OK;
}

int check_table(const char* call, int32_t pt_stride, int32_t n) {
  if (n < 0 || n > QC_KV8_MAX_SEQS)
    return refuse(QC_ERR_ARG, "%s: %d sequences, limit is %d", call, n, QC_KV8_MAX_SEQS);
  if (pt_stride < 1) return refuse(QC_ERR_ARG, "%s: pt_stride %d", call, pt_stride);
  return QC_OK;
}

int rows_call(const char* call, bool write, const qc_kv8_cache* c, const int32_t* table,
              int32_t pt_stride, const int32_t* pos, const int32_t* start, int32_t n, int32_t rows,
              uint16_t* k, int64_t k_ld, uint16_t* v, int64_t v_ld, qc_stream stream) {
  int rc = check_cache(call, c);
  if (rc) return rc;
  if (rows < 0) return refuse(QC_ERR_ARG, "%s: n_rows %d", call, rows);
  if (!start && rows != n)
    return refuse(QC_ERR_ARG, "%s: %d rows for %d sequences without row_start", call, rows, n);
  const int64_t width = int64_t(c->n_kv_heads) * c->head_dim;
  if (k_ld < width || v_ld < width || ((k_ld | v_ld) & 7))
    return refuse(QC_ERR_ARG, "%s: row strides %lld and %lld (multiples of 8, at least %lld)", call,
                  (long long)k_ld, (long long)v_ld, (long long)width);
  if (!aligned16(k) || !aligned16(v))
    return refuse(QC_ERR_ARG, "%s: k and v must be 16-byte aligned", call);
  if (!aligned4(table) || !aligned4(pos) || !aligned4(start))
    return refuse(QC_ERR_ARG, "%s: page table, pos and row_start must be 4-byte aligned", call);
  rc = check_table(call, pt_stride, n);
  if (rc || n == 0 || rows == 0) return rc;
  rc = BufferCheck(call)
           .need("the pool", c->pool)
           .need("page_table_dev", table)
           .need("pos_dev", pos)
           .maybe("row_start_dev", start)
           .need("k_dev", k)
           .need("v_dev", v)
           .check();
  if (rc) return rc;

  Kv8RowsArgs a{};
  a.pool = c->pool;
  a.table = table;
  a.pos = pos;
  a.start = start;
  a.k = k;
  a.v = v;
  a.k_ld = k_ld;
  a.v_ld = v_ld;
  a.n_pages = c->n_pages;
  a.pt_stride = pt_stride;
  a.kv_heads = c->n_kv_heads;
  a.n = n;
  a.rows = rows;
  // every touched block holds a new row, and only a sequence's first and last
  // block can hold fewer than 16
  const int64_t blocks =
      start ? std::min<int64_t>(rows, int64_t(rows) / BT + 2 * int64_t(n)) : int64_t(n);
  const int64_t per_cta = TW / 2 * (256 / c->head_dim);
  const int64_t ctas = (blocks * c->n_kv_heads + per_cta - 1) / per_cta;
  if (ctas * per_cta > 1 << 26)  // over 256 GB of rows
    return refuse(QC_ERR_ARG, "%s: %d rows of %d heads", call, rows, c->n_kv_heads);
  const dim3 grid((unsigned)ctas);
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
#define QC_ROWS(D)                                                                          \
  e = write ? launch_dependent(kv8_rows_kernel<D, true>, grid, 32 * TW, 0, s, a)            \
            : launch_dependent(kv8_rows_kernel<D, false>, grid, 32 * TW, 0, s, a)
  if (c->head_dim == 64) QC_ROWS(64);
  else if (c->head_dim == 128) QC_ROWS(128);
  else QC_ROWS(256);
#undef QC_ROWS
  return e == cudaSuccess ? QC_OK : refuse(QC_ERR_CUDA, "%s: %s", call, cudaGetErrorString(e));
}

}  // namespace
}  // namespace qc

extern "C" int64_t qc_kv8_page_bytes(int32_t n_kv_heads, int32_t head_dim) {
  if (n_kv_heads < 1 || n_kv_heads > QC_KV8_MAX_HEADS ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  return int64_t(n_kv_heads) * qc::PAGE_BLOCKS * qc::block_bytes(head_dim);
}

extern "C" int qc_kv8_write(const qc_kv8_cache* cache, const int32_t* page_table_dev,
                            int32_t pt_stride, const int32_t* pos_dev,
                            const int32_t* row_start_dev, int32_t n, int32_t n_rows,
                            const uint16_t* k_dev, int64_t k_ld, const uint16_t* v_dev,
                            int64_t v_ld, qc_stream stream) {
  qc::TraceRange trace_("qc_kv8_write");
  return qc::rows_call("qc_kv8_write", true, cache, page_table_dev, pt_stride, pos_dev,
                       row_start_dev, n, n_rows, const_cast<uint16_t*>(k_dev), k_ld,
                       const_cast<uint16_t*>(v_dev), v_ld, stream);
}

extern "C" int qc_kv8_read(const qc_kv8_cache* cache, const int32_t* page_table_dev,
                           int32_t pt_stride, const int32_t* pos_dev, const int32_t* row_start_dev,
                           int32_t n, int32_t n_rows, uint16_t* k_dev, int64_t k_ld,
                           uint16_t* v_dev, int64_t v_ld, qc_stream stream) {
  qc::TraceRange trace_("qc_kv8_read");
  return qc::rows_call("qc_kv8_read", false, cache, page_table_dev, pt_stride, pos_dev,
                       row_start_dev, n, n_rows, k_dev, k_ld, v_dev, v_ld, stream);
}

extern "C" int64_t qc_kv8_attn_workspace_bytes(const qc_kv8_cache* cache, int32_t n,
                                               int32_t n_head) {
  if (!cache || !qc_kv8_page_bytes(cache->n_kv_heads, cache->head_dim) || n < 0 ||
      n > QC_KV8_MAX_SEQS || n_head < 1 || n_head % cache->n_kv_heads ||
      n_head / cache->n_kv_heads > QC_KV8_MAX_GROUP)
    return 0;
  return qc::owner_bytes() +
         2 * int64_t(qc::MAX_WARPS) * qc::record_bytes(n_head / cache->n_kv_heads, cache->head_dim);
}

extern "C" int qc_kv8_attn_decode(const qc_kv8_cache* cache, const int32_t* page_table_dev,
                                  int32_t pt_stride, const int32_t* len_dev, int32_t n,
                                  int32_t n_head, const uint16_t* q_dev, int64_t q_ld,
                                  int64_t q_head, const uint16_t* gate_dev, float scale,
                                  uint16_t* out_dev, int64_t out_ld, void* workspace,
                                  int64_t workspace_bytes, qc_stream stream) {
  constexpr const char* CALL = "qc_kv8_attn_decode";
  qc::TraceRange trace_(CALL);
  int rc = qc::check_cache(CALL, cache);
  if (rc) return rc;
  const int32_t kvh = cache->n_kv_heads, dim = cache->head_dim;
  if (n_head < 1 || n_head % kvh || n_head / kvh > QC_KV8_MAX_GROUP)
    return qc::refuse(QC_ERR_ARG, "%s: %d query heads over %d KV heads (1..%d to each)", CALL,
                      n_head, kvh, QC_KV8_MAX_GROUP);
  if ((q_ld | q_head | out_ld) & 7)
    return qc::refuse(QC_ERR_ARG, "%s: strides must be multiples of 8 elements", CALL);
  if (out_ld < int64_t(n_head) * dim && n > 1)
    return qc::refuse(QC_ERR_ARG, "%s: out_ld %lld below %d heads of %d", CALL, (long long)out_ld,
                      n_head, dim);
  if (!qc::aligned16(q_dev) || !qc::aligned16(gate_dev) || !qc::aligned16(out_dev) ||
      !qc::aligned16(workspace))
    return qc::refuse(QC_ERR_ARG, "%s: q, gate, out and workspace must be 16-byte aligned", CALL);
  if (!qc::aligned4(page_table_dev) || !qc::aligned4(len_dev))
    return qc::refuse(QC_ERR_ARG, "%s: page table and len must be 4-byte aligned", CALL);
  rc = qc::check_table(CALL, pt_stride, n);
  if (rc || n == 0) return rc;
  const int64_t need = qc_kv8_attn_workspace_bytes(cache, n, n_head);
  if (workspace_bytes < need)
    return qc::refuse(QC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", CALL,
                      (long long)workspace_bytes, (long long)need);
  rc = qc::BufferCheck(CALL)
           .need("the pool", cache->pool)
           .need("page_table_dev", page_table_dev)
           .need("len_dev", len_dev)
           .need("q_dev", q_dev)
           .maybe("gate_dev", gate_dev)
           .need("out_dev", out_dev)
           .need("workspace", workspace)
           .check();
  if (rc) return rc;

  qc::Kv8AttnArgs a{};
  a.pool = cache->pool;
  a.table = page_table_dev;
  a.len = len_dev;
  a.q = q_dev;
  a.gate = gate_dev;
  a.out = out_dev;
  a.q_ld = q_ld;
  a.q_head = q_head;
  a.out_ld = out_ld;
  a.owner = static_cast<int4*>(workspace);
  a.rec = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + qc::owner_bytes());
  a.scale = std::frexp(scale * 1.44269504088896340736f, &a.scale_exp);  // log2(e): the weights are powers of two
  if (!std::isfinite(a.scale)) a.scale_exp = 0;
  a.n_pages = cache->n_pages;
  a.pt_stride = pt_stride;
  a.kv_heads = kvh;
  a.group = n_head / kvh;
  a.n = n;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  const bool paired = a.group <= 4;
  if (dim == 64) e = paired ? qc::launch_attn<64, true>(a, s) : qc::launch_attn<64, false>(a, s);
  else if (dim == 128) e = paired ? qc::launch_attn<128, true>(a, s) : qc::launch_attn<128, false>(a, s);
  else e = paired ? qc::launch_attn<256, true>(a, s) : qc::launch_attn<256, false>(a, s);
  return e == cudaSuccess ? QC_OK : qc::refuse(QC_ERR_CUDA, "%s: %s", CALL, cudaGetErrorString(e));
}

extern "C" int qc_kv8_check(qc_stream stream) {
  static std::mutex one_at_a_time;  // g_kv8_taken is a check's until it is read
  cudaStream_t s = (cudaStream_t)stream;
  int code = 0;
  cudaError_t e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) {
    std::lock_guard<std::mutex> lock(one_at_a_time);
    e = cudaLaunchKernel(qc::kv8_take_error_kernel, dim3(1), dim3(1), nullptr, 0, s);
    if (e == cudaSuccess)
      e = cudaMemcpyFromSymbolAsync(&code, qc::g_kv8_taken, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
    const cudaError_t done = cudaStreamSynchronize(s);
    if (e == cudaSuccess) e = done;
  }
  if (e != cudaSuccess) return qc::refuse(QC_ERR_CUDA, "qc_kv8_check: %s", cudaGetErrorString(e));
  if (code)
    return qc::refuse(code, "qc_kv8: the device reported %s",
                      code == QC_ERR_BOUNDS ? "a page, position or row out of range (skipped)"
                      : code == QC_ERR_TIMEOUT ? "a wait timeout" : "an error");
  return QC_OK;
}
