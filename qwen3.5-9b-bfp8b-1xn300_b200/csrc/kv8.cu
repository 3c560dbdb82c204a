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

struct Kv8AttnArgs {
  const uint8_t* pool;
  const int32_t *table, *len;
  const uint16_t *q, *gate;
  uint16_t* out;
  int64_t q_ld, q_head, out_ld;
  float scale;
  int32_t n_pages, pt_stride, kv_heads, group, n;
};

// One CTA per (sequence, query head), a block of 16 tokens per warp at a time.
template <int D>
__global__ void __launch_bounds__(256) kv8_attn_kernel(const Kv8AttnArgs a) {
  __shared__ float q[D], o_s[8][D], m_s[8], l_s[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = blockIdx.x, h = blockIdx.y, kvh = h / a.group;
  int64_t len = a.len[seq];
  if (len < 0 || len > int64_t(a.pt_stride) * QC_PAGE) {
    if (tid == 0) record_error(&g_kv8_error, QC_ERR_BOUNDS);
    len = len < 0 ? 0 : int64_t(a.pt_stride) * QC_PAGE;
  }
  for (int d = tid; d < D; d += 256) q[d] = bf2f(a.q[seq * a.q_ld + h * a.q_head + d]);
  __syncthreads();
  const int g = lane >> 2, t = lane & 3, rho = 4 * (g >> 1) + (g & 1);
  float m = -INFINITY, l = 0.0f, o[D / 8] = {};
  for (int64_t b = warp; b * BT < len; b += 8) {
    const int32_t page = a.table[int64_t(seq) * a.pt_stride + b / PAGE_BLOCKS];
    if (page < 0 || page >= a.n_pages) {
      if (lane == 0) record_error(&g_kv8_error, QC_ERR_BOUNDS);
      continue;
    }
    const uint8_t* block =
        a.pool + ((int64_t(page) * a.kv_heads + kvh) * PAGE_BLOCKS + b % PAGE_BLOCKS) * block_bytes(D);
    const float2 sc = *reinterpret_cast<const float2*>(block);
    const int left = int(min(len - b * BT, int64_t(BT)));
    float s[2] = {0.0f, 0.0f};
    for (int i = 0; i < D / 32; ++i) {
      const uint4 w = reinterpret_cast<const uint4*>(block + HEAD_BYTES)[32 * i + lane];
      const uint8_t* c = reinterpret_cast<const uint8_t*>(&w);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[(e >> 2) & 1] += q[32 * i + 16 * (e >> 3) + 4 * t + (e & 3)] * float(int(c[e]) - 128);
    }
    float most = -INFINITY;
    for (int j = 0; j < 2; ++j) {
      s[j] += __shfl_xor_sync(FULL_MASK, s[j], 1);
      s[j] += __shfl_xor_sync(FULL_MASK, s[j], 2);
      s[j] *= sc.x * a.scale;
      if (rho + 2 * j >= left) s[j] = -INFINITY;
      most = fmaxf(most, s[j]);
    }
    most = fmaxf(m, warp_max(most));
    const float keep = expf(m - most);
    m = most;
    l *= keep;
    for (int x = 0; x < D / 8; ++x) o[x] *= keep;
    // weights of tokens 4t .. 4t+3: rows rho = 4t, 4t+1 are at g = 2t, 2t+1
    float p[4];
    for (int j = 0; j < 2; ++j) {
      const float w = rho + 2 * j < left ? expf(s[j] - m) : 0.0f;
      p[2 * j] = __shfl_sync(FULL_MASK, w, (2 * t) * 4);
      p[2 * j + 1] = __shfl_sync(FULL_MASK, w, (2 * t + 1) * 4);
    }
    l += p[0] + p[1] + p[2] + p[3];  // of this t
    for (int i = 0; i < D / 32; ++i) {
      const uint4 w = reinterpret_cast<const uint4*>(block + HEAD_BYTES + BT * D)[32 * i + lane];
      const uint8_t* c = reinterpret_cast<const uint8_t*>(&w);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        for (int e = 0; e < 4; ++e) o[4 * i + x] += p[e] * sc.y * float(int(c[4 * x + e]) - 128);
    }
  }
  l += __shfl_xor_sync(FULL_MASK, l, 1);
  l += __shfl_xor_sync(FULL_MASK, l, 2);
  for (int x = 0; x < D / 8; ++x) {
    o[x] += __shfl_xor_sync(FULL_MASK, o[x], 1);
    o[x] += __shfl_xor_sync(FULL_MASK, o[x], 2);
    if (t == 0) o_s[warp][8 * x + g] = o[x];
  }
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  for (int d = tid; d < D; d += 256) {
    float M = -INFINITY, L = 0.0f, O = 0.0f;
    for (int w = 0; w < 8; ++w) M = fmaxf(M, m_s[w]);
    for (int w = 0; w < 8; ++w) {
      const float f = m_s[w] == -INFINITY ? 0.0f : expf(m_s[w] - M);
      L += l_s[w] * f;
      O += o_s[w][d] * f;
    }
    float y = len > 0 ? O / L : 0.0f;
    if (a.gate && len > 0) y *= sigmoid_exact(bf2f(a.gate[seq * a.q_ld + h * a.q_head + d]));
    a.out[seq * a.out_ld + h * D + d] = f2bf(y);
  }
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
  return 16;
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
  a.scale = scale;
  a.n_pages = cache->n_pages;
  a.pt_stride = pt_stride;
  a.kv_heads = kvh;
  a.group = n_head / kvh;
  a.n = n;
  const dim3 grid((unsigned)n, (unsigned)n_head);
  cudaStream_t s = (cudaStream_t)stream;
  if (dim == 64) qc::kv8_attn_kernel<64><<<grid, 256, 0, s>>>(a);
  else if (dim == 128) qc::kv8_attn_kernel<128><<<grid, 256, 0, s>>>(a);
  else qc::kv8_attn_kernel<256><<<grid, 256, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
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
