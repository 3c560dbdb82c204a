// rope.cu — rotary position embedding of projection rows, with the per-head
// RMSNorm in front of it (include/qrope.h).
//
// One CTA takes one row: its first rot/2 threads work out the row's cosines
// and sines once, for all heads, then every group of lanes takes a head, 8
// dims (16 bytes) a lane.
#include <cmath>
#include <cstring>

#include "../../include/qrope.h"
#include "caller_buffers.h"
#include "common.cuh"
#include "kernels.h"

namespace qc {
namespace {

constexpr int RT = 256;  // threads per CTA

struct RopeArgs {
  double turns[QC_ROPE_MAX_DIM / 2];  // turns per position of each pair: inv_freq / (2 pi)
  qc_rope_part part[QC_ROPE_MAX_PARTS];
  const int32_t* pos;
  float eps, mscale;
  int32_t rows, n_parts, dim, rot, layout;
  int32_t gl;                         // lanes of a head's group: the power of two at or above dim / 8
};

__global__ void __launch_bounds__(RT) rope_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[QC_ROPE_MAX_DIM / 2];
  __shared__ float stage[RT / 32][32 * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = a.gl, sub = lane & (gl - 1);
  const int group = threadIdx.x / gl, groups = RT / gl;
  float* mine = &stage[warp][(lane - sub) * 8];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    if (threadIdx.x < a.rot / 2) {
      // whole turns drop out exactly in 64 bits; what is left is at most half a turn
      const double t = double(a.pos[r]) * a.turns[threadIdx.x];
      float s, c;
      sincospif(float(2.0 * (t - rint(t))), &s, &c);
      cs[threadIdx.x] = make_float2(c * a.mscale, s * a.mscale);
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
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
          for (int m = gl >> 1; m; m >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, m);
          const float rms = 1.0f / sqrtf(ss / float(a.dim) + a.eps);
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
          uint4 y;
          y.x = f2bf(x[0]) | uint32_t(f2bf(x[1])) << 16;
          y.y = f2bf(x[2]) | uint32_t(f2bf(x[3])) << 16;
          y.z = f2bf(x[4]) | uint32_t(f2bf(x[5])) << 16;
          y.w = f2bf(x[6]) | uint32_t(f2bf(x[7])) << 16;
          *reinterpret_cast<uint4*>(q.out + r * q.out_ld + h * q.out_head + sub * 8) = y;
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
    if (q.n_heads < 1) return qc::refuse(QC_ERR_ARG, "%s: n_heads %d", CALL, q.n_heads);
    if ((q.x_ld | q.x_head | q.out_ld | q.out_head) & 7)
      return bad("strides must be multiples of 8 elements");
    if (((uintptr_t)q.x | (uintptr_t)q.out | (uintptr_t)q.norm_w) & 15)
      return bad("x, out and norm_w must be 16-byte aligned");
  }
  if (n_rows == 0) return QC_OK;
  int rc = qc::check_device_pointer(CALL, "pos_dev", pos_dev);
  for (int p = 0; p < n_parts && !rc; ++p) {
    rc = qc::check_device_pointer(CALL, "x", parts[p].x);
    if (!rc) rc = qc::check_device_pointer(CALL, "out", parts[p].out);
    if (!rc && parts[p].norm_w) rc = qc::check_device_pointer(CALL, "norm_w", parts[p].norm_w);
  }
  if (rc) return rc;

  qc::RopeArgs a{};
  for (int i = 0; i < rope->rot_dim / 2; ++i)
    a.turns[i] = rope->inv_freq[i] / (2.0 * 3.14159265358979323846);
  for (int p = 0; p < n_parts; ++p) a.part[p] = parts[p];
  a.pos = pos_dev;
  a.eps = eps;
  a.mscale = float(rope->mscale);
  a.rows = n_rows;
  a.n_parts = n_parts;
  a.dim = head_dim;
  a.rot = rope->rot_dim;
  a.layout = rope->layout;
  a.gl = 1;
  while (a.gl * 8 < head_dim) a.gl *= 2;
  qc::rope_kernel<<<n_rows, qc::RT, 0, (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return qc::refuse(QC_ERR_CUDA, "%s: %s", CALL, cudaGetErrorString(e));
  return QC_OK;
}
