// rope.cu — rotary position embedding of projection rows, with the per-head
// RMSNorm in front of it (include/qrope.h).
//
// Bound by memory: every value is read and written once, and little is done
// with it.  A lane of a row's group owns four pairs for the whole row (rotated
// dims) or 8 dims (the rest), so it works out its four cosines and sines once,
// keeps them in registers over all heads that it takes, and no lane needs
// another's values except for the norm's sum.  32768 rows of 40 heads of 128 (671
// MB) take 113 us, 5.94 TB/s, 0.90 of the measured copy rate; an earlier form, a
// CTA per row with the pairs exchanged through shared memory, took 416 us: too few
// loads in flight behind its barriers.  With the norm an SM issues an instruction in
// two cycles of three (2048 rows of 20 heads of 256: 11.8 us, 6.4 by its bytes).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/qrope.h"
#include "caller_buffers.h"
#include "common.cuh"
#include "kernels.h"

namespace qc {
namespace {

constexpr int RT = 128;   // threads per CTA
struct RopeArgs {
  double turns[QC_ROPE_MAX_DIM / 2];  // turns per position of each pair: inv_freq / (2 pi)
  qc_rope_part part[QC_ROPE_MAX_PARTS];
  int32_t slices[QC_ROPE_MAX_PARTS];  // of `chunk` heads
  const int32_t* pos;
  float eps, mscale, inv_dim;
  int32_t rows, n_parts, dim, rot, layout;
  int32_t gl, gl_log2;                // lanes of a row's group: the power of two at or above dim / 8
  int32_t chunk;                      // heads that a group takes
};

// cos and sin of 2 pi t, t = pos * turns: whole turns drop out exactly in 64
// bits, and what is left is at most half a turn.
__device__ __forceinline__ float2 rotation(const RopeArgs& a, int32_t pos, int pair) {
  const double t = double(pos) * a.turns[pair];
  float s, c;
  sincospif(float(2.0 * (t - rint(t))), &s, &c);
  return make_float2(c * a.mscale, s * a.mscale);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The norm's factor 1 / sqrt(mean(y^2) + eps) of a group's head, of which this lane has
// 8 dims; all lanes of the warp call it.  Where the squares leave f32 (values beyond
// 1.8e19, or all below 3e-14 with as small an eps) y is first brought to about 1 by a
// power of two, exactly but for what is 2^-126 of the head's largest value.  The vote on
// that costs 0.6 us of the 11.8 of 2048 rows of 20 heads of 256; one vote for four heads,
// or a loop of their own for such heads, costs as much or more, in registers.
__device__ __forceinline__ float norm_factor(const RopeArgs& a, float (&y)[8]) {
  const auto mean = [&](float eps) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
    for (int m = a.gl >> 1; m; m >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, m);
    return ss * a.inv_dim + eps;
  };
  float v = mean(a.eps);
  const bool odd = !(v >= 0x1p-90f && v < INFINITY);
  if (__any_sync(FULL_MASK, odd)) {
    float top = sqrtf(a.eps);  // eps * down^2 must not leave f32 either
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[e]));
    for (int m = a.gl >> 1; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, m));
    const int at = int(__float_as_uint(top) >> 23);  // 255: an infinity, the sum shows it
    const float down = odd && top > 0.0f && at < 255 ? __uint_as_float(uint32_t(max(254 - at, 1)) << 23) : 1.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= down;
    v = mean(a.eps * down * down);
  }
  return rsqrtf(v);
}

// rot_dim a multiple of 8.  gl lanes take a row's heads h0 .. h1-1 of one part
// (blockIdx.y); lane j holds pairs 4j .. 4j+3 for j < rot / 8 — in the half
// layout two runs of 4 dims, 4j and rot/2 + 4j, in the interleaved one 8 dims in
// a row — and dims 8j .. 8j+7 from there on.  RU heads' loads go out before the
// first is used, and before the angles are worked out.
template <bool HALF, bool NORM, int RU>
__global__ void __launch_bounds__(RT) rope_kernel(const __grid_constant__ RopeArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int p = 0, slice = blockIdx.y;
  while (slice >= a.slices[p]) slice -= a.slices[p++];
  const qc_rope_part& q = a.part[p];
  const int h0 = slice * a.chunk, h1 = min(h0 + a.chunk, int(q.n_heads));
  const int gl = a.gl, j = threadIdx.x & (gl - 1);
  const int64_t r = (int64_t(blockIdx.x) * RT + threadIdx.x) >> a.gl_log2;
  const bool on = r < a.rows && 8 * j < a.dim, turn = on && 8 * j < a.rot;
  // this lane's two runs of 4 dims
  const int da = HALF && turn ? 4 * j : 8 * j, db = HALF && turn ? a.rot / 2 + 4 * j : 8 * j + 4;
  const bool wide = !(HALF && turn);
  const uint16_t* src = q.x + r * q.x_ld + h0 * q.x_head;
  uint16_t* dst = q.out + r * q.out_ld + h0 * q.out_head;
  const int32_t pos = turn ? a.pos[r] : 0;
  float w[8];
  const bool norm = NORM && q.norm_w;
  if (norm && on) {
    const float4 wa = *reinterpret_cast<const float4*>(q.norm_w + da);
    const float4 wb = *reinterpret_cast<const float4*>(q.norm_w + db);
    w[0] = wa.x; w[1] = wa.y; w[2] = wa.z; w[3] = wa.w;
    w[4] = wb.x; w[5] = wb.y; w[6] = wb.z; w[7] = wb.w;
  }
  float2 cs[4];
  // every group makes the same number of turns: those of one warp meet in the norm's shuffles
  for (int h = h0; h < h0 + a.chunk; h += RU) {
    uint4 x[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      x[u] = make_uint4(0, 0, 0, 0);
      if (on && h + u < h1) {
        if (wide) {
          x[u] = *reinterpret_cast<const uint4*>(src + da);
        } else {
          const uint2 lo = *reinterpret_cast<const uint2*>(src + da);
          const uint2 hi = *reinterpret_cast<const uint2*>(src + db);
          x[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        src += q.x_head;
      }
    }
    if (turn && h == h0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[e] = rotation(a, pos, 4 * j + e);
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      float y[8];
      unpack8(x[u], y);
      if (norm) {
        const float rms = norm_factor(a, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * rms * w[e];
      }
      if (turn) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i1 = HALF ? e : 2 * e, i2 = HALF ? e + 4 : 2 * e + 1;
          const float y1 = y[i1], y2 = y[i2];
          y[i1] = y1 * cs[e].x - y2 * cs[e].y;
          y[i2] = y2 * cs[e].x + y1 * cs[e].y;
        }
      }
      if (on && h + u < h1) {
        const uint4 z = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]),
                                   pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
        if (wide) {
          *reinterpret_cast<uint4*>(dst + da) = z;
        } else {
          *reinterpret_cast<uint2*>(dst + da) = make_uint2(z.x, z.y);
          *reinterpret_cast<uint2*>(dst + db) = make_uint2(z.z, z.w);
        }
        dst += q.out_head;
      }
    }
  }
}

// Any even rot_dim: a CTA per row, pairs exchanged through shared memory.
__global__ void __launch_bounds__(RT) rope_any_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[QC_ROPE_MAX_DIM / 2];
  __shared__ float stage[RT / 32][32 * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = a.gl, sub = lane & (gl - 1);
  const int group = threadIdx.x / gl, groups = RT / gl;
  float* mine = &stage[warp][(lane - sub) * 8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    if (threadIdx.x < a.rot / 2) {
      cs[threadIdx.x] = rotation(a, a.pos[r], threadIdx.x);
    }
    __syncthreads();
    for (int p = 0; p < a.n_parts; ++p) {
      const qc_rope_part& q = a.part[p];
      // every lane of a warp makes the same number of turns, so that the shuffles meet
      for (int h0 = 0; h0 < q.n_heads; h0 += groups) {
        const int h = h0 + group;
        const bool on = h < q.n_heads && sub * 8 < a.dim;
        float x[8] = {};
        if (on) unpack8(*reinterpret_cast<const uint4*>(q.x + r * q.x_ld + h * q.x_head + sub * 8), x);
        if (q.norm_w) {
          const float rms = norm_factor(a, x);
          if (on) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * rms * q.norm_w[sub * 8 + e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[sub * 8 + e] = x[e];
        __syncwarp();
        if (on) {
          const int half = a.rot / 2;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = sub * 8 + e;
            if (d >= a.rot) continue;
            if (a.layout == QC_ROPE_HALF) {
              const bool low = d < half;
              const float2 w = cs[low ? d : d - half];
              const float o = mine[low ? d + half : d - half];
              x[e] = low ? x[e] * w.x - o * w.y : x[e] * w.x + o * w.y;
            } else {
              const float2 w = cs[d / 2];
              const float o = mine[d ^ 1];
              x[e] = d & 1 ? x[e] * w.x + o * w.y : x[e] * w.x - o * w.y;
            }
          }
          *reinterpret_cast<uint4*>(q.out + r * q.out_ld + h * q.out_head + sub * 8) =
              make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]),
                         pack_bf16(x[6], x[7]));
        }
        __syncwarp();
      }
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace qc

extern "C" int qc_rope_init(const qc_rope_config* cfg, qc_rope* rope) {
  constexpr const char* CALL = "qc_rope_init";
  auto bad = [&](const char* why) { return qc::refuse(QC_ERR_ARG, "%s: %s", CALL, why); };
  if (!cfg || !rope) return bad("null argument");
  const int rot = cfg->rot_dim;
  if (rot < 2 || rot > QC_ROPE_MAX_DIM || rot % 2)
    return bad("rot_dim is not an even number in [2, 256]");
  if (cfg->layout != QC_ROPE_HALF && cfg->layout != QC_ROPE_INTERLEAVED)
    return bad("unknown layout");
  if (cfg->scaling < QC_ROPE_PLAIN || cfg->scaling > QC_ROPE_YARN)
    return bad("unknown scaling");
  if (!(cfg->base > 1.0) || !std::isfinite(cfg->base)) return bad("base must be above 1");
  const bool scaled = cfg->scaling != QC_ROPE_PLAIN, yarn = cfg->scaling == QC_ROPE_YARN;
  if (scaled && (!(cfg->factor > 0.0) || !std::isfinite(cfg->factor)))
    return bad("factor must be above 0");
  if (cfg->scaling == QC_ROPE_NTK && rot == 2) return bad("NTK scaling needs rot_dim above 2");
  if (!std::isfinite(cfg->mscale) || cfg->mscale < 0.0) return bad("mscale must be 0 or above");
  const double fast = cfg->beta_fast == 0.0 ? 32.0 : cfg->beta_fast;
  const double slow = cfg->beta_slow == 0.0 ? 1.0 : cfg->beta_slow;
  if (yarn && (cfg->orig_ctx < 1 || !(fast > 0.0) || !(slow > 0.0) || !std::isfinite(fast) ||
               !std::isfinite(slow)))
    return bad("YARN needs orig_ctx and both betas above 0");

  const double pi = 3.14159265358979323846;
  double base = cfg->base, low = 0.0, high = 0.0;
  if (cfg->scaling == QC_ROPE_NTK) base *= std::pow(cfg->factor, double(rot) / (rot - 2));
  if (yarn) {
    // the pair index at which a frequency makes b turns within the trained context
    auto turn = [&](double b) {
      return rot * std::log(cfg->orig_ctx / (b * 2.0 * pi)) / (2.0 * std::log(base));
    };
    low = std::fmax(std::floor(turn(fast)), 0.0);
    high = std::fmin(std::ceil(turn(slow)), rot - 1.0);
  }
  qc_rope r;
  std::memset(&r, 0, sizeof(r));
  r.rot_dim = rot;
  r.layout = cfg->layout;
  r.mscale = cfg->mscale != 0.0                  ? cfg->mscale
             : yarn && cfg->factor > 1.0 ? 0.1 * std::log(cfg->factor) + 1.0
                                                 : 1.0;
  for (int i = 0; i < rot / 2; ++i) {
    const double w = std::pow(base, -2.0 * i / rot);
    if (cfg->scaling == QC_ROPE_LINEAR) {
      r.inv_freq[i] = w / cfg->factor;
    } else if (yarn) {
      const double g = std::fmin(std::fmax((i - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
      r.inv_freq[i] = w / cfg->factor * g + w * (1.0 - g);
    } else {
      r.inv_freq[i] = w;
    }
    if (!std::isfinite(r.inv_freq[i])) return bad("base and factor give an infinite frequency");
  }
  *rope = r;
  return QC_OK;
}

extern "C" int qc_rope_apply(const qc_rope* rope, int32_t head_dim, float eps,
                             const int32_t* pos_dev, int32_t n_rows, const qc_rope_part* parts,
                             int32_t n_parts, qc_stream stream) {
  constexpr const char* CALL = "qc_rope_apply";
  auto bad = [&](const char* why) { return qc::refuse(QC_ERR_ARG, "%s: %s", CALL, why); };
  qc::TraceRange trace_("qc_rope_apply");
  if (!rope || !parts) return bad("null argument");
  if (rope->rot_dim < 2 || rope->rot_dim > QC_ROPE_MAX_DIM || rope->rot_dim % 2 ||
      (rope->layout != QC_ROPE_HALF && rope->layout != QC_ROPE_INTERLEAVED))
    return bad("not a struct that qc_rope_init filled");
  if (head_dim < 8 || head_dim % 8 || head_dim > QC_ROPE_MAX_DIM || rope->rot_dim > head_dim)
    return qc::refuse(QC_ERR_ARG, "%s: head_dim %d with rot_dim %d", CALL, head_dim, rope->rot_dim);
  if (n_rows < 0) return qc::refuse(QC_ERR_ARG, "%s: n_rows %d", CALL, n_rows);
  if (n_parts < 1 || n_parts > QC_ROPE_MAX_PARTS)
    return qc::refuse(QC_ERR_ARG, "%s: n_parts %d", CALL, n_parts);
  if (!(eps >= 0.0f)) return bad("eps must be 0 or above");
  for (int p = 0; p < n_parts; ++p) {
    const qc_rope_part& q = parts[p];
    if (q.n_heads < 1 || q.n_heads > QC_ROPE_MAX_HEADS)
      return qc::refuse(QC_ERR_ARG, "%s: n_heads %lld", CALL, (long long)q.n_heads);
    if ((q.x_ld | q.x_head | q.out_ld | q.out_head) & 7)
      return bad("strides must be multiples of 8 elements");
    if (((uintptr_t)q.x | (uintptr_t)q.out | (uintptr_t)q.norm_w) & 15)
      return bad("x, out and norm_w must be 16-byte aligned");
  }
  if (!qc::aligned4(pos_dev)) return bad("pos_dev must be 4-byte aligned");
  if (n_rows == 0) return QC_OK;
  qc::BufferCheck buffers(CALL);
  buffers.need("pos_dev", pos_dev);
  for (int p = 0; p < n_parts; ++p)
    buffers.need("x", parts[p].x).need("out", parts[p].out).maybe("norm_w", parts[p].norm_w);
  if (buffers.check()) return buffers.check();

  qc::RopeArgs a{};
  for (int i = 0; i < rope->rot_dim / 2; ++i)
    a.turns[i] = rope->inv_freq[i] / (2.0 * 3.14159265358979323846);
  for (int p = 0; p < n_parts; ++p) a.part[p] = parts[p];
  a.pos = pos_dev;
  a.eps = eps;
  a.inv_dim = 1.0f / float(head_dim);
  a.mscale = float(rope->mscale);
  a.rows = n_rows;
  a.n_parts = n_parts;
  a.dim = head_dim;
  a.rot = rope->rot_dim;
  a.layout = rope->layout;
  a.gl = 1;
  while (a.gl * 8 < head_dim) {
    a.gl *= 2;
    ++a.gl_log2;
  }
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (a.rot % 8) {
    e = qc::launch_dependent(qc::rope_any_kernel, dim3(n_rows), qc::RT, 0, s, a);
  } else {
    bool norm = false;
    int32_t most = 1;
    for (int p = 0; p < n_parts; ++p) {
      norm |= parts[p].norm_w != nullptr;
      most = std::max(most, int32_t(parts[p].n_heads));
    }
    // A group takes as many of its row's heads as leave WANT threads (two waves of
    // each of a B200's 148 SMs), as each group works out the row's angles again: 2048 and
    // 4096 rows of 20 normalised heads of 256 take 11.8 and 20.6 us so, 12.7 and 25.9 with
    // half as many threads.  With fewer than FEW threads one head to a group is faster,
    // the others' loads and arithmetic being latency alone: 8 rows 1.9 against 3.2 us, 64
    // rows 2.7 and 3.3, 128 rows 3.2 and 3.6; 1024 rows 10.0 and 6.6.
    auto slices = [&](int32_t chunk) {
      int32_t n = 0;
      for (int p = 0; p < n_parts; ++p) n += a.slices[p] = (int32_t(parts[p].n_heads) + chunk - 1) / chunk;
      return n;
    };
    constexpr int64_t WANT = 148 * 2048, FEW = 148 * 256;
    a.chunk = (most + 3) / 4 * 4;
    while (a.chunk > 4 && int64_t(n_rows) * a.gl * slices(a.chunk) < WANT)
      a.chunk = (a.chunk / 2 + 3) / 4 * 4;
    const bool few = int64_t(n_rows) * a.gl * slices(a.chunk) < FEW && slices(1) < 65536;
    if (few) a.chunk = 1;
    const dim3 grid((unsigned)((int64_t(n_rows) * a.gl + qc::RT - 1) / qc::RT),
                    (unsigned)slices(a.chunk));
    const bool half = rope->layout == QC_ROPE_HALF;
#define QC_ROPE(H, N)                                                                       \
  e = few ? qc::launch_dependent(qc::rope_kernel<H, N, 1>, grid, qc::RT, 0, s, a)           \
          : qc::launch_dependent(qc::rope_kernel<H, N, 4>, grid, qc::RT, 0, s, a)
    if (half && norm) QC_ROPE(true, true);
    else if (half) QC_ROPE(true, false);
    else if (norm) QC_ROPE(false, true);
    else QC_ROPE(false, false);
#undef QC_ROPE
  }
  if (e != cudaSuccess) return qc::refuse(QC_ERR_CUDA, "%s: %s", CALL, cudaGetErrorString(e));
  return QC_OK;
}
