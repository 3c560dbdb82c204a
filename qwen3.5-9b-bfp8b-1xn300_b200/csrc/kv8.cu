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

// First error of these kernels on this device since the last qc_kv8_check.
__device__ int g_kv8_error;

struct Kv8RowsArgs {
  uint8_t* pool;
  const int32_t *table, *pos, *start;  // start null: one row each
  uint16_t *k, *v;
  int64_t k_ld, v_ld;
  int32_t n_pages, pt_stride, kv_heads, n, rows;
};

__device__ __forceinline__ int64_t blocks_touched(int64_t pos, int64_t cnt) {
  return cnt > 0 ? (pos + cnt - 1) / BT - pos / BT + 1 : 0;
}

// bf16 bits as the value that is quantised: NaN is 0, what 127 * 2^120 does not
// reach saturates there.
__device__ __forceinline__ float storable(uint16_t b) {
  const float x = bf2f(b);
  const float most = 0x1.FCp+126f;  // 127 * 2^120
  return x != x ? 0.0f : fminf(fmaxf(x, -most), most);
}

// The smallest power of two s with amax <= 127 s, at least 2^-126.  With amax =
// 1.M * 2^(E - 127) that is 2^(E - 133), or twice it when 1.M > 127 / 64.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = int(u >> 23) - 133 + ((u & 0x7fffffu) > 0x7e0000u);
  e = max(e, -126);
  return __uint_as_float(uint32_t(e + 127) << 23);
}

__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return uint32_t(__float2int_rn(fminf(fmaxf(x * inv, -127.0f), 127.0f)) + 128);
}

// One CTA of D threads per (touched block, kv head); warp i holds dims 32 i ..
// 32 i + 31 and each thread the 16 bytes of K and of V that it also writes.
template <int D, bool WRITE>
__global__ void __launch_bounds__(D) kv8_rows_kernel(const Kv8RowsArgs a) {
  __shared__ int64_t found[2];
  __shared__ int64_t sums[D];
  __shared__ float amax_s[2][D / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y;

  // which sequence and which of its blocks this CTA is: the blocks of all
  // sequences, counted in order
  if (a.start) {
    int64_t base = 0;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    for (int i0 = 0; i0 < a.n; i0 += D) {
      const int i = i0 + tid;
      int64_t nb = 0;
      if (i < a.n) {
        const int64_t cnt = int64_t(a.start[i + 1]) - a.start[i];
        nb = a.pos[i] < 0 ? 0 : blocks_touched(a.pos[i], cnt);
        if (a.pos[i] < 0 && cnt > 0) record_error(&g_kv8_error, QC_ERR_BOUNDS);
      }
      sums[tid] = nb;
      __syncthreads();
      for (int m = 1; m < D; m <<= 1) {
        const int64_t add = tid >= m ? sums[tid - m] : 0;
        __syncthreads();
        sums[tid] += add;
        __syncthreads();
      }
      const int64_t begin = base + sums[tid] - nb, b = blockIdx.x;
      if (b >= begin && b < begin + nb) {
        found[0] = i;
        found[1] = b - begin;
      }
      base += sums[D - 1];
      __syncthreads();
    }
    // rows that overlap or leave the input can ask for more blocks than there are CTAs
    if (tid == 0 && base > int64_t(gridDim.x)) record_error(&g_kv8_error, QC_ERR_BOUNDS);
  } else if (tid == 0) {
    found[0] = blockIdx.x;
    found[1] = 0;
    if (a.pos[blockIdx.x] < 0) {
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
      found[0] = -1;
    }
  }
  __syncthreads();
  const int seq = int(found[0]);
  if (seq < 0) return;
  const int64_t first = a.pos[seq];
  const int64_t row0 = a.start ? a.start[seq] : seq;
  const int64_t cnt = a.start ? a.start[seq + 1] - row0 : 1;
  const int64_t begin = (first / BT + found[1]) * BT;          // first position of the block
  const int lo = first > begin ? int(first - begin) : 0;       // new rows of the block: [lo, hi)
  const int hi = int(min(first + cnt - begin, int64_t(BT)));
  const int64_t row_of = row0 + begin - first;                 // input row of slot 0
  const int64_t pg = begin / QC_PAGE;
  const int32_t page = pg < a.pt_stride ? a.table[int64_t(seq) * a.pt_stride + pg] : -1;
  if (page < 0 || page >= a.n_pages || row_of + lo < 0 || row_of + hi > a.rows) {
    if (tid == 0) record_error(&g_kv8_error, QC_ERR_BOUNDS);
    return;
  }
  uint8_t* block = a.pool + ((int64_t(page) * a.kv_heads + head) * PAGE_BLOCKS + begin % QC_PAGE / BT) *
                                block_bytes(D);
  uint4* kc = reinterpret_cast<uint4*>(block + HEAD_BYTES) + tid;
  uint4* vc = kc + D;  // 16 * D bytes further
  const int g = lane >> 2, t = lane & 3;
  const int rho = 4 * (g >> 1) + (g & 1);
  // slot and dim of byte e of this thread's 16 K bytes and of its 16 V bytes
  auto k_slot = [&](int e) { return rho + 2 * ((e >> 2) & 1); };
  auto k_dim = [&](int e) { return 32 * warp + 16 * (e >> 3) + 4 * t + (e & 3); };
  auto v_slot = [&](int e) { return 4 * t + (e & 3); };
  auto v_dim = [&](int e) { return 32 * warp + 16 * (e >> 3) + 8 * ((e >> 2) & 1) + g; };

  if (!WRITE) {
    const float2 sc = *reinterpret_cast<const float2*>(block);
    const uint4 kw = *kc, vw = *vc;
    const uint8_t* kb = reinterpret_cast<const uint8_t*>(&kw);
    const uint8_t* vb = reinterpret_cast<const uint8_t*>(&vw);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (k_slot(e) >= lo && k_slot(e) < hi)
        a.k[(row_of + k_slot(e)) * a.k_ld + head * D + k_dim(e)] = f2bf(float(int(kb[e]) - 128) * sc.x);
      if (v_slot(e) >= lo && v_slot(e) < hi)
        a.v[(row_of + v_slot(e)) * a.v_ld + head * D + v_dim(e)] = f2bf(float(int(vb[e]) - 128) * sc.y);
    }
    return;
  }

  float kx[16], vx[16], ka = 0.0f, va = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    kx[e] = vx[e] = 0.0f;
    if (k_slot(e) >= lo && k_slot(e) < hi)
      kx[e] = storable(a.k[(row_of + k_slot(e)) * a.k_ld + head * D + k_dim(e)]);
    if (v_slot(e) >= lo && v_slot(e) < hi)
      vx[e] = storable(a.v[(row_of + v_slot(e)) * a.v_ld + head * D + v_dim(e)]);
    ka = fmaxf(ka, fabsf(kx[e]));
    va = fmaxf(va, fabsf(vx[e]));
  }
  ka = warp_max(ka);
  va = warp_max(va);
  if (lane == 0) {
    amax_s[0][warp] = ka;
    amax_s[1][warp] = va;
  }
  // the block's scales before this call are read before anything is written
  const float2 old = *reinterpret_cast<const float2*>(block);
  __syncthreads();
  for (int w = 0; w < D / 32; ++w) {
    ka = fmaxf(ka, amax_s[0][w]);
    va = fmaxf(va, amax_s[1][w]);
  }
  float ks = pow2_scale(ka), vs = pow2_scale(va);
  if (lo > 0) {  // older tokens stay: the scale does not shrink
    ks = fmaxf(ks, old.x);
    vs = fmaxf(vs, old.y);
  }
  if (tid == 0) *reinterpret_cast<float2*>(block) = make_float2(ks, vs);
  const float ki = 1.0f / ks, vi = 1.0f / vs;
  const float kr = old.x / ks, vr = old.y / vs;
  const bool whole = lo == 0 && hi == BT;
  uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
  if (!whole) {
    kw = *kc;
    vw = *vc;
  }
  uint8_t* kb = reinterpret_cast<uint8_t*>(&kw);
  uint8_t* vb = reinterpret_cast<uint8_t*>(&vw);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    if (k_slot(e) < lo) kb[e] = uint8_t(code_of(float(int(kb[e]) - 128) * kr, 1.0f));
    else if (k_slot(e) < hi) kb[e] = uint8_t(code_of(kx[e], ki));
    if (v_slot(e) < lo) vb[e] = uint8_t(code_of(float(int(vb[e]) - 128) * vr, 1.0f));
    else if (v_slot(e) < hi) vb[e] = uint8_t(code_of(vx[e], vi));
  }
  *kc = kw;
  *vc = vw;
}

// ---------------------------------------------------------------- attention
//
// out = sum_j 2^(x_j - m) V_j / sum_j 2^(x_j - m), x_j = scale * log2(e) q.K_j,
// one pass over the blocks with a running maximum.
//
// Split.  The blocks of all (sequence, kv head) pairs, counted in order, are cut
// into one equal contiguous range per warp of the grid.  A warp streams its
// blocks through its own ring of bulk copies (one of 16 + 32 D bytes a block:
// scales, K, V) and works on each alone: no barrier joins warps.  A pair that
// lies whole in one range is finished there; of the others every range writes a
// record (m, l, r, o), which the combine kernel merges in order.
//
// Products.  S = K q on m16n8k16 f16 with f32 sums: the codes are whole numbers
// up to 127 and the bf16 queries, scaled by a power of two, are exact in f16, so
// the products are exact.  Two byte permutes and two subtractions turn four
// codes into f16: byte u under 0x64 is 1024 + u, less 1152 the code.  The row
// order of the cache makes S, transposed by movmatrix, the operand of
// O^T = V^T w without any other exchange.
//
// The weights of the second product carry V's scale: w = 2^(x + log2 sv - r)
// with a running reference r of its own, so blocks of very different scales
// keep their precision (l has no part in it).  w stands in f16, at most 2^15;
// groups of up to 4 heads use the product's other 4 columns for w - f16(w), so
// that 22 bits of it count.  Both references move only when a score passes them
// by 2^8 (m; r starts 2^7 under its largest and moves at 2^15), so most blocks
// rescale nothing.

struct Kv8AttnArgs {
  const uint8_t* pool;
  const int32_t *table, *len;
  const uint16_t *q, *gate;
  uint16_t* out;
  int4* owner;      // a split pair: sequence, kv head, its number of records, the first of them;
                    // one entry per pair (by_pair) or for the last pair that each warp starts
  float* rec;       // [warps][2][group][D + 4]: m, l, r, unused, o
  int64_t q_ld, q_head, out_ld;
  float scale;      // scale * log2(e)
  int32_t n_pages, pt_stride, kv_heads, group, n;
  int32_t by_pair;
};

constexpr int AW = 4;                                    // warps per CTA
constexpr int AS = 3;                                    // blocks in flight per warp
constexpr int MIN_BLOCKS = 1;                            // blocks of a warp's range at least
constexpr int MAX_WARPS = 2400;                          // of the grid
constexpr float LAZY_M = 8.0f, TOP_R = 7.0f, LAZY_R = 15.0f;

template <int D>
struct AttnSmem {
  alignas(128) uint8_t stage[AW][AS][block_bytes(D)];
  alignas(8) uint64_t full[AW][AS];
  int32_t valid[AW][AS];                                 // tokens of the block; 0: nothing was copied
  int64_t sums[AW + 1];
  struct { int64_t unit; int32_t seq; } start[AW];       // first unit of the sequence a warp starts in
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

__device__ __forceinline__ int64_t seq_blocks(const Kv8AttnArgs& a, int32_t i) {
  const int64_t most = int64_t(a.pt_stride) * QC_PAGE;
  return (min(max(int64_t(a.len[i]), int64_t(0)), most) + BT - 1) / BT;
}

// Where in the order of blocks a warp stands: `unit` counts the blocks of all
// pairs, `blk` those of the pair (seq, head), which has nb.
struct Cursor {
  int64_t unit;
  int32_t seq, head, blk, nb, len;

  __device__ __forceinline__ void enter(const Kv8AttnArgs& a) {
    nb = int32_t(seq_blocks(a, seq));
    len = int32_t(min(int64_t(a.len[seq]), int64_t(a.pt_stride) * QC_PAGE));
  }
  // To the next pair that has blocks; the caller knows that there is one.
  __device__ __forceinline__ void next_pair(const Kv8AttnArgs& a) {
    blk = 0;
    if (++head == a.kv_heads) {
      head = 0;
      do {
        ++seq;
      } while (seq + 1 < a.n && seq_blocks(a, seq) == 0);
      enter(a);
    }
  }
};

template <int D, bool PAIRED>
__global__ void __launch_bounds__(32 * AW) kv8_attn_kernel(const Kv8AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  AttnSmem<D>& sm = *reinterpret_cast<AttnSmem<D>*>(smem_raw);
  constexpr int KS = D / 16;  // steps of 16 dims
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < AS; ++s) mbar_init(&sm.full[w][s], 1);
    fence_mbar_init();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Blocks before each sequence: thread i sums its run of sequences, the runs
  // are scanned, and the threads whose run holds a warp's first block say so.
  const int warps = gridDim.x * AW, wid = w * gridDim.x + blockIdx.x;
  const int run = (a.n + 32 * AW - 1) / (32 * AW);
  int64_t mine = 0;
  for (int j = 0; j < run; ++j) {
    const int i = tid * run + j;
    if (i < a.n) {
      const int64_t nb = seq_blocks(a, i);
      mine += nb;
      if (blockIdx.x == 0 && (a.len[i] < 0 || a.len[i] > int64_t(a.pt_stride) * QC_PAGE))
        record_error(&g_kv8_error, QC_ERR_BOUNDS);
      // a sequence without tokens has a row of zeros and nothing to merge
      if (nb == 0 && i % int(gridDim.x) == int(blockIdx.x)) {
        for (int d = 0; d < a.kv_heads * a.group * D; d += 8)
          *reinterpret_cast<uint4*>(a.out + i * a.out_ld + d) = make_uint4(0, 0, 0, 0);
        for (int h = 0; h < a.kv_heads && a.by_pair; ++h)
          a.owner[i * a.kv_heads + h] = make_int4(0, 0, 0, 0);
      }
    }
  }
  int64_t before = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t x = __shfl_up_sync(FULL_MASK, before, m);
    if (lane >= m) before += x;
  }
  if (lane == 31) sm.sums[w] = before;
  __syncthreads();
  int64_t total = 0;
  before -= mine;
  for (int x = 0; x < AW; ++x) {
    if (x < w) before += sm.sums[x];
    total += sm.sums[x];
  }
  total *= a.kv_heads;
  before *= a.kv_heads;
  const int64_t per = max((total + warps - 1) / warps, int64_t(MIN_BLOCKS));
  for (int x = 0; x < AW; ++x) {
    const int64_t u = (int64_t(x) * gridDim.x + blockIdx.x) * per;
    if (u >= before && u < before + mine * a.kv_heads) {
      int64_t at = before;
      for (int j = 0; j < run; ++j) {
        const int64_t nb = seq_blocks(a, tid * run + j) * a.kv_heads;
        if (u < at + nb) {
          sm.start[x].unit = at;
          sm.start[x].seq = tid * run + j;
          break;
        }
        at += nb;
      }
    }
  }
  __syncthreads();
  const int64_t begin = wid * per, end = min(begin + per, total);
  if (lane == 0 && !a.by_pair) a.owner[wid] = make_int4(0, 0, 0, 0);
  if (begin >= end) return;

  Cursor c;
  c.unit = begin;
  c.seq = sm.start[w].seq;
  c.enter(a);
  c.head = int32_t((begin - sm.start[w].unit) / c.nb);
  c.blk = int32_t((begin - sm.start[w].unit) % c.nb);
  Cursor p = c;  // the copies run AS blocks ahead
  int put = 0;
  auto issue = [&]() {  // lane 0: the copy of block p into the next stage
    if (p.unit >= end) return;
    const int32_t page = __ldg(a.table + int64_t(p.seq) * a.pt_stride + p.blk / PAGE_BLOCKS);
    const bool ok = page >= 0 && page < a.n_pages;
    sm.valid[w][put] = ok ? min(p.len - p.blk * BT, BT) : 0;
    if (ok) {
      mbar_arrive_expect_tx(&sm.full[w][put], block_bytes(D));
      bulk_g2s(sm.stage[w][put],
               a.pool + ((int64_t(page) * a.kv_heads + p.head) * PAGE_BLOCKS + p.blk % PAGE_BLOCKS) *
                            block_bytes(D),
               block_bytes(D), &sm.full[w][put]);
    } else {
      record_error(&g_kv8_error, QC_ERR_BOUNDS);
      mbar_arrive(&sm.full[w][put]);
    }
    put = put + 1 == AS ? 0 : put + 1;
    ++p.unit;
    if (++p.blk == p.nb && p.unit < end) p.next_pair(a);
  };
  if (lane == 0)
    for (int s = 0; s < AS; ++s) issue();

  int get = 0;
  uint32_t parity = 0;
  bool first = true;
  while (c.unit < end) {
    // ---- the pair's queries, as operand columns: column n is head n (PAIRED: n % 4)
    const int32_t blk0 = c.blk;
    uint32_t qf[KS][2];
    float qs[2];  // what a column's products count for: scale log2(e) / the power of two in q
    {
      const int h = PAIRED ? g & 3 : g;
      uint2 raw[KS];
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        raw[s] = make_uint2(0, 0);
        if (h < a.group)
          raw[s] = *reinterpret_cast<const uint2*>(
              a.q + c.seq * a.q_ld + (int64_t(c.head) * a.group + h) * a.q_head + 16 * s + 4 * t);
        // bf16 magnitudes order as their bits
        top = max(top, max(max(raw[s].x & 0x7fffu, (raw[s].x >> 16) & 0x7fffu),
                           max(raw[s].y & 0x7fffu, (raw[s].y >> 16) & 0x7fffu)));
      }
      top = max(top, __shfl_xor_sync(FULL_MASK, top, 1));
      top = max(top, __shfl_xor_sync(FULL_MASK, top, 2));
      // up * 2^e: the largest value into [2^13, 2^14), so that values 2^-37 of it stay exact
      const int e = max(int(top >> 7) - 127 - 13, -126);
      const float up = __uint_as_float(uint32_t(127 - e) << 23);
      float back = a.scale * __uint_as_float(uint32_t(127 + e) << 23);
      if (top >= 0x7f80u) back = __uint_as_float(0x7fc00000u);  // the whole row is NaN
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bool odd = top >= 0x7f80u;
        qf[s][0] = odd ? 0u : pack_f16(bf_lo(raw[s].x) * up, bf_hi(raw[s].x) * up);
        qf[s][1] = odd ? 0u : pack_f16(bf_lo(raw[s].y) * up, bf_hi(raw[s].y) * up);
      }
      qs[0] = __shfl_sync(FULL_MASK, back, 8 * t);
      qs[1] = __shfl_sync(FULL_MASK, back, 8 * t + 4);
    }
    float m[2] = {-INFINITY, -INFINITY}, r[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[KS][4];
#pragma unroll
    for (int s = 0; s < KS; ++s) o[s][0] = o[s][1] = o[s][2] = o[s][3] = 0.0f;

    const int32_t stop = int32_t(min(int64_t(c.nb), c.blk + (end - c.unit)));
    for (; c.blk < stop; ++c.blk, ++c.unit) {
      if (!mbar_wait(&sm.full[w][get], parity, &g_kv8_error)) {
        // leave nothing in flight: the other copies of this warp, each again bounded
        for (int s = 0; s < AS; ++s) {
          const int x = get + s < AS ? get + s : get + s - AS;
          if (c.unit + s < end) mbar_wait(&sm.full[w][x], get + s < AS ? parity : parity ^ 1, nullptr);
        }
        return;
      }
      const int valid = sm.valid[w][get];
      const uint8_t* block = sm.stage[w][get];
      if (valid > 0) {
        const float2 sc = *reinterpret_cast<const float2*>(block);
        const uint4* kc = reinterpret_cast<const uint4*>(block + HEAD_BYTES) + lane;
        const uint4* vc = kc + D;
        float acc[2][4] = {};
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
          const uint4 x = kc[32 * i];
          mma_f16(acc[0], codes_lo(x.x), codes_lo(x.y), codes_hi(x.x), codes_hi(x.y), qf[2 * i][0],
                  qf[2 * i][1]);
          mma_f16(acc[1], codes_lo(x.z), codes_lo(x.w), codes_hi(x.z), codes_hi(x.w),
                  qf[2 * i + 1][0], qf[2 * i + 1][1]);
        }
        // acc[.][0], [1]: token rho, columns 2t, 2t + 1; [2], [3]: token rho + 2
        const int rho = 4 * (g >> 1) + (g & 1);
        const float lsv = float(int((__float_as_uint(sc.y) >> 23) & 0xffu) - 127);
        float x[4];
        bool move = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = (acc[0][j] + acc[1][j]) * qs[j & 1] * sc.x;
          if (rho + (j & 2) >= valid) x[j] = -INFINITY;
          move |= x[j] > m[j & 1] + LAZY_M || x[j] + lsv > r[j & 1] + LAZY_R;
        }
        if (__any_sync(FULL_MASK, move)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = fmaxf(x[j], x[j + 2]);
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 4));
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 8));
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 16));
            const float m1 = fmaxf(m[j], top), r1 = fmaxf(r[j], top + lsv - TOP_R);
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
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = rho + (j & 2) < valid;
          l[j & 1] += in ? ex2(x[j] - m[j & 1]) : 0.0f;
          y[j] = in ? ex2(x[j] + lsv - r[j & 1]) : 0.0f;
          if (PAIRED && t >= 2) y[j] -= __half2float(__float2half_rn(y[j]));
        }
        const uint32_t b0 = transpose8(pack_f16(y[0], y[1]));
        const uint32_t b1 = transpose8(pack_f16(y[2], y[3]));
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
          const uint4 v = vc[32 * i];
          mma_f16(o[2 * i], codes_lo(v.x), codes_lo(v.y), codes_hi(v.x), codes_hi(v.y), b0, b1);
          mma_f16(o[2 * i + 1], codes_lo(v.z), codes_lo(v.w), codes_hi(v.z), codes_hi(v.w), b0, b1);
        }
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0) issue();
      get = get + 1 == AS ? 0 : get + 1;
      if (get == 0) parity ^= 1;
    }

    // ---- the pair's result, or its record
    const bool done = c.blk == c.nb, whole = done && blk0 == 0;
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
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int h = 2 * t + j;  // o[.][j]: dim g of the 16, o[.][j + 2]: dim g + 8
      if (h >= a.group) continue;
      if (whole) {
        // o 2^(r - m) / l, the power in two halves: either alone may leave f32
        const float half = 0.5f * (r[j] - m[j]);
        const float f1 = l[j] == 0.0f ? 0.0f : ex2(half) / l[j];
        const float f2 = l[j] == 0.0f ? 0.0f : ex2(r[j] - m[j] - half);
        const int64_t head = int64_t(c.head) * a.group + h;
        uint16_t* out = a.out + c.seq * a.out_ld + head * D;
        const uint16_t* gate = a.gate ? a.gate + c.seq * a.q_ld + head * a.q_head : nullptr;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int d = 16 * s + 8 * k + g;
            float y = o[s][j + 2 * k] * f1 * f2;
            if (gate) y *= sigmoid_exact(bf2f(gate[d]));
            out[d] = f2bf(y);
          }
      } else {
        float* rec = a.rec + ((int64_t(wid) * 2 + (first ? 0 : 1)) * a.group + h) * (D + 4);
        if (g == 0) *reinterpret_cast<float4*>(rec) = make_float4(m[j], l[j], r[j], 0.0f);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) rec[4 + 16 * s + 8 * k + g] = o[s][j + 2 * k];
      }
    }
    // the range that a pair starts in says what there is to merge
    if (lane == 0 && blk0 == 0 && (!done || a.by_pair)) {
      const int64_t last = (c.unit - c.blk + c.nb - 1) / per;
      a.owner[a.by_pair ? c.seq * a.kv_heads + c.head : wid] =
          make_int4(c.seq, c.head, done ? 0 : int(last) - wid + 1, 2 * wid + (first ? 0 : 1));
    }
    first = false;
    if (done && c.unit < end) c.next_pair(a);
  }
}

// Merges the records of a split pair: CTA (owner entry, head of the group, CHUNK
// dims), CHUNK / 4 lanes across the dims and the rest of the 256 threads along
// the records, which are the owner's and then the first ones of the warps after
// it.  One pass over the records' heads gives the references and sums, a second
// adds the o in order.
template <int D, int CHUNK>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Kv8AttnArgs a) {
  constexpr int LANES = CHUNK / 4, SLOTS = 256 / LANES;
  __shared__ float4 part[SLOTS][LANES];
  __shared__ float fac[MAX_WARPS];
  __shared__ float2 top_s[8];
  __shared__ float sum_s[8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int4 own = a.owner[blockIdx.x];
  const int n = min(own.z, MAX_WARPS);
  if (n == 0) return;
  const int64_t step = int64_t(a.group) * (D + 4);
  auto rec = [&](int i) {
    return a.rec + (i == 0 ? own.w : 2 * (own.w / 2 + i)) * step + h * (D + 4);
  };
  const int64_t head = int64_t(own.y) * a.group + h;
  const int dim = CHUNK * blockIdx.z + tid;
  float gate = 0.0f;
  if (a.gate && tid < CHUNK) gate = bf2f(a.gate[own.x * a.q_ld + head * a.q_head + dim]);
  float m = -INFINITY, r = -INFINITY, l = 0.0f;
  for (int i = tid; i < n; i += 256) {
    const float4 s = *reinterpret_cast<const float4*>(rec(i));
    // l under the running m; it is 0 exactly where a record met no token, NaN passes
    const float m1 = fmaxf(m, s.x);
    if (s.y != 0.0f) l = l * (l == 0.0f ? 1.0f : ex2(m - m1)) + s.y * (s.x == m1 ? 1.0f : ex2(s.x - m1));
    m = m1;
    r = fmaxf(r, s.z);
    fac[i] = s.y == 0.0f ? -INFINITY : s.z;
  }
  const float mw = warp_max(m), rw = warp_max(r);
  if (lane == 0) top_s[w] = make_float2(mw, rw);
  __syncthreads();
  float M = -INFINITY;
  for (int x = 0; x < 8; ++x) {
    M = fmaxf(M, top_s[x].x);
    r = fmaxf(r, top_s[x].y);
  }
  l = warp_sum(l == 0.0f || m == M ? l : l * ex2(m - M));
  if (lane == 0) sum_s[w] = l;
  const int quad = tid % LANES, slot = tid / LANES;
  float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
  for (int i = slot; i < n; i += SLOTS) {
    const float f = fac[i] == r ? 1.0f : ex2(fac[i] - r);
    const float4 x = *reinterpret_cast<const float4*>(rec(i) + 4 + CHUNK * blockIdx.z + 4 * quad);
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  }
  part[slot][quad] = o;
  __syncthreads();
  if (tid < CHUNK) {
    float y = 0.0f, total = 0.0f;
    for (int x = 0; x < 8; ++x) total += sum_s[x];
    for (int s = 0; s < SLOTS; ++s) y += reinterpret_cast<const float*>(part[s])[tid];
    const float half = 0.5f * (r - M);
    y = total == 0.0f ? 0.0f : y * (ex2(half) / total) * ex2(r - M - half);
    if (a.gate) y *= sigmoid_exact(gate);
    a.out[own.x * a.out_ld + head * D + dim] = f2bf(y);
  }
}

// Workspace: owners of MAX_WARPS warps, then their records.
int64_t owner_bytes() { return int64_t(MAX_WARPS) * sizeof(int4); }
int64_t record_bytes(int32_t group, int32_t dim) { return int64_t(group) * (dim + 4) * sizeof(float); }

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
    grid = std::max(1, std::min(sms * per, MAX_WARPS / AW));
    if (dev < 64) ctas[dev].store(grid, std::memory_order_relaxed);
    configured.mark(dev);
  }
  const int warps = grid * AW;
  const int64_t pairs = int64_t(a.n) * a.kv_heads;
  a.by_pair = pairs <= warps;
  const int entries = a.by_pair ? int(pairs) : warps;
  e = launch_dependent(kv8_attn_kernel<D, PAIRED>, dim3(grid), 32 * AW, sizeof(AttnSmem<D>), s, a);
  if (e != cudaSuccess) return e;
  // few heads have many records each: then 64 dims to a CTA, 16 threads along them
  if (entries * a.group <= 256)
    return launch_dependent(kv8_merge_kernel<D, 64>, dim3(entries, a.group, D / 64), 256, 0, s, a);
  return launch_dependent(kv8_merge_kernel<D, D>, dim3(entries, a.group, 1), 256, 0, s, a);
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

int check_table(const char* call, const qc_kv8_cache* c, const int32_t* table, int32_t pt_stride,
                int32_t n) {
  if (n < 0 || n > QC_KV8_MAX_SEQS)
    return refuse(QC_ERR_ARG, "%s: %d sequences, limit is %d", call, n, QC_KV8_MAX_SEQS);
  if (pt_stride < 1) return refuse(QC_ERR_ARG, "%s: pt_stride %d", call, pt_stride);
  if (n == 0) return QC_OK;
  const int rc = check_device_pointer(call, "the pool", c->pool);
  return rc ? rc : check_device_pointer(call, "page_table_dev", table);
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
  rc = check_table(call, c, table, pt_stride, n);
  if (rc) return rc;
  if (n == 0 || rows == 0) return QC_OK;
  if ((rc = check_device_pointer(call, "pos_dev", pos))) return rc;
  if (start && (rc = check_device_pointer(call, "row_start_dev", start))) return rc;
  if ((rc = check_device_pointer(call, "k_dev", k))) return rc;
  if ((rc = check_device_pointer(call, "v_dev", v))) return rc;

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
  const int64_t most = std::min<int64_t>(rows, int64_t(rows) / BT + 2 * int64_t(n));
  const dim3 grid(start ? (unsigned)most : (unsigned)n, (unsigned)c->n_kv_heads);
  cudaStream_t s = (cudaStream_t)stream;
#define QC_ROWS(D)                                                      \
  if (write) kv8_rows_kernel<D, true><<<grid, D, 0, s>>>(a);            \
  else kv8_rows_kernel<D, false><<<grid, D, 0, s>>>(a)
  if (c->head_dim == 64) { QC_ROWS(64); }
  else if (c->head_dim == 128) { QC_ROWS(128); }
  else { QC_ROWS(256); }
#undef QC_ROWS
  const cudaError_t e = cudaGetLastError();
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
  rc = qc::check_table(CALL, cache, page_table_dev, pt_stride, n);
  if (rc || n == 0) return rc;
  const int64_t need = qc_kv8_attn_workspace_bytes(cache, n, n_head);
  if (workspace_bytes < need)
    return qc::refuse(QC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", CALL,
                      (long long)workspace_bytes, (long long)need);
  if ((rc = qc::check_device_pointer(CALL, "len_dev", len_dev))) return rc;
  if ((rc = qc::check_device_pointer(CALL, "q_dev", q_dev))) return rc;
  if (gate_dev && (rc = qc::check_device_pointer(CALL, "gate_dev", gate_dev))) return rc;
  if ((rc = qc::check_device_pointer(CALL, "out_dev", out_dev))) return rc;
  if ((rc = qc::check_device_pointer(CALL, "workspace", workspace))) return rc;

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
  a.scale = scale * 1.44269504088896340736f;  // log2(e): the weights are powers of two
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
  cudaError_t e = cudaStreamSynchronize((cudaStream_t)stream);
  int code = 0;
  const int zero = 0;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&code, qc::g_kv8_error, sizeof(int));
  if (e == cudaSuccess && code) e = cudaMemcpyToSymbol(qc::g_kv8_error, &zero, sizeof(int));
  if (e != cudaSuccess) return qc::refuse(QC_ERR_CUDA, "qc_kv8_check: %s", cudaGetErrorString(e));
  if (code)
    return qc::refuse(code, "qc_kv8: the device reported %s",
                      code == QC_ERR_BOUNDS ? "a page, position or row out of range (skipped)"
                      : code == QC_ERR_TIMEOUT ? "a wait timeout" : "an error");
  return QC_OK;
}
