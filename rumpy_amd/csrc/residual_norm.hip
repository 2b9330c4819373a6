// The joint between two residual blocks in one pass over the rows: the norm behind a block, its gate, the residual scale, the skip, and the
// norm in front of the next block,
//   z = N_post(t) ;  y = x + scale * g * z ;  h = N_pre(y)            (rows = pixels of an NHWC tensor, or tokens; C channels)
//   N(v) = (v - mean) / sqrt(var + eps) * w + b   ('layer')   |   v / sqrt(mean(v^2) + eps) * w + b   ('rms')   |   v   (none)
// and its backward pass
//   a = dh w ; dY = dy + rs_y (a - mean(a) - yhat mean(a yhat)) ; dx = dY ; dw = sum dh yhat ; db = sum dh
//   dg = scale z dY (summed over the rows a gate row serves) ; dz = scale g dY ; dwp = sum dz that ; dbp = sum dz
//   dt = rs_t (dz wp - mean(dz wp) - that mean(dz wp that))                                    (rms: no mean(.) term)
// About 16 / 34 flops per element against 8 / 12 bytes (16-bit tensors): bound by memory, so each tensor is touched once per direction and
// everything between load and store stays in registers.  A row is spread over TPR lanes, 8 channels (one 16-byte access) each: up to 512
// channels a row stays inside a wave (no barrier), beyond it a workgroup holds one row and joins its waves' sums through LDS.  y is made
// again in the backward pass from x and t instead of being read: the same number of bytes, and the unrounded y (so that h's gradient is that of
// the h that was stored, which the forward pass also took from the unrounded y).  The mean and the factor of each norm are kept per row (fp32).
// Column sums (parameters, gates) run in a fixed order: registers over a workgroup's contiguous rows, one partial row per workgroup, then
// residual_norm_reduce_kernel - bitwise reproducible, no atomics.
#include "row_vec.hpp"

constexpr int RN_GATE_NONE = 0, RN_GATE_GROUP = 1, RN_GATE_FULL = 2;
constexpr int RN_NONE = 0, RN_LAYER = 1, RN_RMS = 2;
constexpr int RN_MAXC = 8192;

// sums over the TPR lanes of a row; rows of more than a wave meet in LDS.  `par` alternates between two buffers, so one barrier per call is enough:
// a wave that writes a buffer again has passed the barrier of the call in between, which every wave enters after its last read of that buffer.
template <int TPR> struct RowSum {
  static constexpr int WAVES = TPR <= 64 ? 1 : TPR / 64;
  float (*buf)[2 * WAVES];
  int par;
  __device__ __forceinline__ void two(float& a, float& b) {
    const int lane = threadIdx.x & 63;
    a = lanes_sum<(TPR < 64 ? TPR : 64)>(a, lane);
    b = lanes_sum<(TPR < 64 ? TPR : 64)>(b, lane);
    if constexpr (WAVES > 1) {
      const int w = threadIdx.x >> 6;
      if (lane == 0) { buf[par][w] = a; buf[par][WAVES + w] = b; }
      __syncthreads();
      float sa = 0.f, sb = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) { sa += buf[par][i]; sb += buf[par][WAVES + i]; }
      a = sa; b = sb;
      par ^= 1;
    }
  }
  __device__ __forceinline__ float one(float a) { float b = 0.f; two(a, b); return a; }
};

__device__ __forceinline__ void load_params(const float* p, int col, int n, float dflt, float (&o)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (p && i < n) ? p[col + i] : dflt;
}

// mean and 1 / sqrt(var + eps) of a row whose elements lie n per lane (zero beyond n)
template <int TPR> __device__ __forceinline__ void row_stats(RowSum<TPR>& sum, const float (&v)[8], int n, int kind, float inv_c, float eps, float& mu, float& rs) {
  mu = 0.f;
  if (kind == RN_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
    mu = sum.one(s) * inv_c;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) { const float d = i < n ? v[i] - mu : 0.f; q = fmaf(d, d, q); }
  rs = 1.f / sqrtf(sum.one(q) * inv_c + eps);
}

template <int XF, int TF, int TPR> __global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR) residual_norm_fwd_kernel(rumpy_residual_norm_args a) {
  constexpr int WG = TPR <= 64 ? 256 : TPR, SUB = WG / TPR;
  __shared__ float red[2][2 * RowSum<TPR>::WAVES];
  RowSum<TPR> sum{red, 0};
  const int tid = threadIdx.x, col = (tid % TPR) * 8, sub = tid / TPR;
  const int nc = min(8, max(0, a.C - col));
  const float inv_c = 1.f / (float)a.C;
  float wp[8], bp[8], w[8], b[8];
  load_params(a.post_w, col, nc, 1.f, wp);
  load_params(a.post_b, col, nc, 0.f, bp);
  load_params(a.pre_w, col, nc, 1.f, w);
  load_params(a.pre_b, col, nc, 0.f, b);
  for (int64_t rb = (int64_t)blockIdx.x * SUB; rb < a.rows; rb += (int64_t)gridDim.x * SUB) {
    const int64_t r = rb + sub;
    const bool live = r < a.rows;                   // (a row of more than a wave: always)
    const int n = live ? nc : 0;
    const size_t rr = live ? (size_t)r : 0;
    float y[8];
    load8<XF>(a.x, rr * a.ldx + col, n, y);
    float mu = 0.f, rs = 1.f;
    if (a.t) {
      float t[8], g[8];
      load8<TF>(a.t, rr * a.ldt + col, n, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = 1.f;
      if (a.gate_mode == RN_GATE_GROUP) load_params((const float*)a.gate + (size_t)((uint32_t)rr / (uint32_t)a.group_rows) * a.C, col, n, 0.f, g);
      else if (a.gate_mode == RN_GATE_FULL) load8<TF>(a.gate, rr * a.ldg + col, n, g);
      if (a.post != RN_NONE) row_stats<TPR>(sum, t, n, a.post, inv_c, a.eps, mu, rs);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = fmaf((t[i] - mu) * rs, wp[i], bp[i]);
        y[i] = i < n ? fmaf(a.scale * g[i], z, y[i]) : 0.f;
      }
      store8<XF>(a.y, rr * a.C + col, n, y);
      if (a.stats && a.post != RN_NONE && live && col == 0) { a.stats[rr] = mu; a.stats[a.rows + rr] = rs; }
    }
    if (a.pre != RN_NONE) {
      row_stats<TPR>(sum, y, n, a.pre, inv_c, a.eps, mu, rs);
      float h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = fmaf((y[i] - mu) * rs, w[i], b[i]);
      store8<TF>(a.h, rr * a.C + col, n, h);
      if (a.stats && live && col == 0) { a.stats[2 * a.rows + rr] = mu; a.stats[3 * a.rows + rr] = rs; }
    }
  }
}

// ---- backward ----
// Work of one launch: `wgs` workgroups of `rpw` contiguous rows each.  A gate row that serves a group of rows is summed over a workgroup's part
// of the group and stored as partial row (workgroup + group): over the walk of all (workgroup, group) pairs that number grows strictly.  Groups
// shorter than a workgroup's step store one partial row per row instead.
struct RnPlan { int tpr, sub, wgs, rpw; bool direct; };
static RnPlan rn_plan(int64_t rows, int64_t group_rows, int32_t C, int gate_mode) {
  RnPlan p;
  p.tpr = 8;
  while (p.tpr * 8 < C) p.tpr *= 2;
  p.sub = p.tpr <= 64 ? 256 / p.tpr : 1;
  const int64_t steps = (rows + p.sub - 1) / p.sub;
  int64_t wgs = (steps + 3) / 4;
  if (wgs > 512) wgs = 512;
  if (wgs < 1) wgs = 1;
  p.rpw = (int)((steps + wgs - 1) / wgs * p.sub);
  p.wgs = (int)((rows + p.rpw - 1) / p.rpw);
  p.direct = gate_mode == RN_GATE_GROUP && group_rows < p.sub;
  return p;
}

// column sums of a workgroup: the rows of a step lie side by side in its waves
template <int TPR> __device__ __forceinline__ void flush_columns(float (&acc)[8], float* dst, int col, int nc, float* lds) {
  if constexpr (TPR > 64) {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < nc) dst[col + i] = acc[i];
  } else {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = acc[i];
#pragma unroll
      for (int o = TPR; o < 64; o *= 2) v += __shfl_xor(v, o);
      acc[i] = v;
    }
    __syncthreads();
    if (lane < TPR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) lds[wave * TPR * 8 + lane * 8 + i] = acc[i];
    }
    __syncthreads();
    if (tid < TPR) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < nc) dst[col + i] = (lds[tid * 8 + i] + lds[TPR * 8 + tid * 8 + i]) + (lds[2 * TPR * 8 + tid * 8 + i] + lds[3 * TPR * 8 + tid * 8 + i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
}

template <int XF, int TF, int TPR> __global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR) residual_norm_bwd_kernel(rumpy_residual_norm_bwd_args a, RnPlan plan) {
  constexpr int WG = TPR <= 64 ? 256 : TPR, SUB = WG / TPR;
  __shared__ float red[2][2 * RowSum<TPR>::WAVES];
  __shared__ float cols[TPR <= 64 ? 4 * TPR * 8 : 1];
  RowSum<TPR> sum{red, 0};
  const int tid = threadIdx.x, col = (tid % TPR) * 8, sub = tid / TPR;
  const int nc = min(8, max(0, a.C - col));
  const float inv_c = 1.f / (float)a.C;
  float wp[8], bp[8], w[8], g[8];
  load_params(a.post_w, col, nc, 1.f, wp);
  load_params(a.post_b, col, nc, 0.f, bp);
  load_params(a.pre_w, col, nc, 1.f, w);
  float aw[8], ab[8], awp[8], abp[8], ag[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { aw[i] = ab[i] = awp[i] = abp[i] = ag[i] = 0.f; g[i] = 1.f; }
  const int64_t r0 = (int64_t)blockIdx.x * plan.rpw, r1 = min(a.rows, r0 + plan.rpw);
  float* part = a.partial;                                            // [4][wgs][C], then the gate's partial rows
  float* gpart = a.partial + (size_t)4 * plan.wgs * a.C;
  const bool group_sums = a.gate_mode == RN_GATE_GROUP && !plan.direct;
  for (int64_t seg = r0; seg < r1;) {
    int64_t seg_end = r1;
    size_t group = 0;
    if (group_sums) {
      group = (uint32_t)seg / (uint32_t)a.group_rows;
      seg_end = min(r1, (int64_t)(group + 1) * a.group_rows);
      load_params((const float*)a.gate + group * a.C, col, nc, 0.f, g);
    }
    for (int64_t rb = seg; rb < seg_end; rb += SUB) {
      const int64_t r = rb + sub;
      const bool live = r < seg_end;
      const int n = live ? nc : 0;
      const size_t rr = live ? (size_t)r : (size_t)seg;
      float x[8], t[8], d[8], e[8];
      load8<XF>(a.x, rr * a.ldx + col, n, x);
      if (a.t) load8<TF>(a.t, rr * a.ldt + col, n, t);
      if (a.dy) load8<XF>(a.dy, rr * a.lddy + col, n, d);
      else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
      }
      if (a.dh) load8<TF>(a.dh, rr * a.lddh + col, n, e);
      if (a.gate_mode == RN_GATE_FULL) load8<TF>(a.gate, rr * a.ldg + col, n, g);
      else if (plan.direct) load_params((const float*)a.gate + (size_t)((uint32_t)rr / (uint32_t)a.group_rows) * a.C, col, n, 0.f, g);
      float mu_t = 0.f, rs_t = 1.f;
      if (a.t) {
        if (a.post != RN_NONE) { mu_t = a.stats[rr]; rs_t = a.stats[a.rows + rr]; }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[i] = i < n ? (t[i] - mu_t) * rs_t : 0.f;                                // that
          x[i] = i < n ? fmaf(a.scale * g[i], fmaf(t[i], wp[i], bp[i]), x[i]) : 0.f;     // y, unrounded
        }
      }
      if (a.dh) {
        const float mu = a.stats[2 * a.rows + rr], rs = a.stats[3 * a.rows + rr];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float yh = i < n ? (x[i] - mu) * rs : 0.f;
          x[i] = yh;
          ab[i] += e[i];
          aw[i] = fmaf(e[i], yh, aw[i]);
          e[i] *= w[i];
          s1 += e[i];
          s2 = fmaf(e[i], yh, s2);
        }
        sum.two(s1, s2);
        s1 = a.pre == RN_LAYER ? s1 * inv_c : 0.f;
        s2 *= inv_c;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = fmaf(rs, (e[i] - s1) - x[i] * s2, d[i]);
      }
      if (a.dx) store8<XF>(a.dx, rr * a.C + col, n, d);
      if (!a.t) continue;
      float s1 = 0.f, s2 = 0.f;
      float gr[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float dd = i < n ? a.scale * d[i] : 0.f;
        gr[i] = dd * fmaf(t[i], wp[i], bp[i]);
        ag[i] += gr[i];
        const float dz = g[i] * dd;
        abp[i] += dz;
        awp[i] = fmaf(dz, t[i], awp[i]);
        d[i] = dz * wp[i];
        s1 += d[i];
        s2 = fmaf(d[i], t[i], s2);
      }
      if (a.gate_mode == RN_GATE_FULL) { if (a.dgate) store8<TF>(a.dgate, rr * a.C + col, n, gr); }
      else if (plan.direct && a.dgate) store8<RUMPY_FMT_F32>(gpart, rr * a.C + col, n, gr);
      if (a.post != RN_NONE) {
        sum.two(s1, s2);
        s1 = a.post == RN_LAYER ? s1 * inv_c : 0.f;
        s2 *= inv_c;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = rs_t * ((d[i] - s1) - t[i] * s2);
      }
      if (a.dt) store8<TF>(a.dt, rr * a.C + col, n, d);
    }
    if (group_sums && a.dgate) flush_columns<TPR>(ag, gpart + (blockIdx.x + group) * a.C, col, nc, cols);
    seg = seg_end;
  }
  const size_t wc = (size_t)plan.wgs * a.C;
  float* mine = part + (size_t)blockIdx.x * a.C;
  if (a.d_post_w) flush_columns<TPR>(awp, mine, col, nc, cols);
  if (a.d_post_b) flush_columns<TPR>(abp, mine + wc, col, nc, cols);
  if (a.d_pre_w) flush_columns<TPR>(aw, mine + 2 * wc, col, nc, cols);
  if (a.d_pre_b) flush_columns<TPR>(ab, mine + 3 * wc, col, nc, cols);
}

// out[c] = sum over consecutive partial rows: items 0..3 = the parameters (all workgroups), 4.. = the gate rows
__global__ void __launch_bounds__(256) residual_norm_reduce_kernel(rumpy_residual_norm_bwd_args a, RnPlan plan, int tiles) {
  __shared__ float red[4][64];
  const size_t item = blockIdx.x / tiles;
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6, c = (blockIdx.x % tiles) * 64 + lane;
  const size_t wc = (size_t)plan.wgs * a.C;
  const float* src;
  float* dst;
  int64_t count;
  if (item < 4) {
    float* const outs[4] = {a.d_post_w, a.d_post_b, a.d_pre_w, a.d_pre_b};
    dst = outs[item];
    src = a.partial + item * wc;
    count = plan.wgs;
  } else {
    const int64_t group = (int64_t)item - 4, first = group * a.group_rows, last = min(a.rows, first + a.group_rows) - 1;
    dst = a.dgate ? (float*)a.dgate + group * a.C : nullptr;
    src = a.partial + 4 * wc;
    if (plan.direct) { src += (size_t)first * a.C; count = last - first + 1; }
    else { const int64_t w0 = first / plan.rpw, w1 = last / plan.rpw; src += (size_t)(w0 + group) * a.C; count = w1 - w0 + 1; }
  }
  if (!dst) return;                                            // (the whole workgroup)
  float s = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int64_t i = slice; i < count; i += 4) s += src[(size_t)i * a.C + c];
  }
  red[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < a.C) dst[c] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// ---- entry points ----
static bool rn_formats_ok(int x_fmt, int t_fmt) {
  return (x_fmt == t_fmt && (x_fmt == RUMPY_FMT_F32 || x_fmt == RUMPY_FMT_BF16 || x_fmt == RUMPY_FMT_F16)) ||
         (x_fmt == RUMPY_FMT_F32 && (t_fmt == RUMPY_FMT_BF16 || t_fmt == RUMPY_FMT_F16));
}
// what both directions have in common; returns a message or nullptr
static const char* rn_check(int64_t rows, int64_t group_rows, int32_t C, int x_fmt, int t_fmt, const void* t, const void* gate, int gate_mode, int post, int pre) {
  if (rows < 0 || rows > 0x7fffffff) return "0 .. 2^31 - 1 rows";
  if (C < 1 || C > RN_MAXC) return "1 .. 8192 channels";
  if (!rn_formats_ok(x_fmt, t_fmt)) return "x and the branch in one format, or x in fp32 beside a 16-bit branch";
  if (post < RN_NONE || post > RN_RMS || pre < RN_NONE || pre > RN_RMS) return "norm kinds 0 .. 2";
  if (gate_mode < RN_GATE_NONE || gate_mode > RN_GATE_FULL || (gate_mode != RN_GATE_NONE) != (gate != nullptr)) return "gate modes 0 .. 2, with the gate's pointer";
  if (!t && (post != RN_NONE || gate_mode != RN_GATE_NONE || pre == RN_NONE)) return "without a branch there is only the norm in front";
  if (gate_mode == RN_GATE_GROUP && (group_rows < 1 || group_rows > 0x7fffffff || rows % group_rows)) return "a gate row serves a whole number of rows";
  return nullptr;
}

template <int XF, int TF> static void rn_launch_fwd(const rumpy_residual_norm_args& a, const RnPlan& p, hipStream_t s) {
  const int64_t steps = (a.rows + p.sub - 1) / p.sub;
  const dim3 grid((unsigned)(steps < 4096 ? steps : 4096));
  switch (p.tpr) {
    case 8: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 8>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 16>), grid, dim3(256), 0, s, a); break;
    case 32: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 32>), grid, dim3(256), 0, s, a); break;
    case 64: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 64>), grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 128>), grid, dim3(128), 0, s, a); break;
    case 256: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 256>), grid, dim3(256), 0, s, a); break;
    case 512: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 512>), grid, dim3(512), 0, s, a); break;
    default: hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, 1024>), grid, dim3(1024), 0, s, a); break;
  }
}
template <int XF, int TF> static void rn_launch_bwd(const rumpy_residual_norm_bwd_args& a, const RnPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.wgs);
  switch (p.tpr) {
    case 8: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 8>), grid, dim3(256), 0, s, a, p); break;
    case 16: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 16>), grid, dim3(256), 0, s, a, p); break;
    case 32: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 32>), grid, dim3(256), 0, s, a, p); break;
    case 64: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 64>), grid, dim3(256), 0, s, a, p); break;
    case 128: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 128>), grid, dim3(128), 0, s, a, p); break;
    case 256: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 256>), grid, dim3(256), 0, s, a, p); break;
    case 512: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 512>), grid, dim3(512), 0, s, a, p); break;
    default: hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, 1024>), grid, dim3(1024), 0, s, a, p); break;
  }
}
#define RN_BY_FORMAT(fn, ...)                                                                                          \
  do {                                                                                                                 \
    if (p->x_fmt == RUMPY_FMT_BF16) fn<RUMPY_FMT_BF16, RUMPY_FMT_BF16>(__VA_ARGS__);                                    \
    else if (p->x_fmt == RUMPY_FMT_F16) fn<RUMPY_FMT_F16, RUMPY_FMT_F16>(__VA_ARGS__);                                  \
    else if (p->t_fmt == RUMPY_FMT_BF16) fn<RUMPY_FMT_F32, RUMPY_FMT_BF16>(__VA_ARGS__);                                \
    else if (p->t_fmt == RUMPY_FMT_F16) fn<RUMPY_FMT_F32, RUMPY_FMT_F16>(__VA_ARGS__);                                  \
    else fn<RUMPY_FMT_F32, RUMPY_FMT_F32>(__VA_ARGS__);                                                                \
  } while (0)

extern "C" int rumpy_residual_norm_fwd(const rumpy_residual_norm_args* p, void* stream) {
  const char* bad = !p ? "no arguments" : rn_check(p->rows, p->group_rows, p->C, p->x_fmt, p->t_fmt, p->t, p->gate, p->gate_mode, p->post, p->pre);
  if (!bad && p->rows && (!p->x || (p->t && !p->y) || (p->pre != RN_NONE && !p->h))) bad = "a tensor is missing";
  if (!bad && (p->ldx < 0 || p->ldt < 0 || p->ldg < 0)) bad = "row strides are not negative";
  if (bad) { rumpy_set_error("rumpy_residual_norm_fwd: %s", bad); return RUMPY_E_ARG; }
  if (p->rows == 0) return RUMPY_OK;
  const RnPlan plan = rn_plan(p->rows, p->group_rows, p->C, p->gate_mode);
  RN_BY_FORMAT(rn_launch_fwd, *p, plan, (hipStream_t)stream);
  return rumpy_check_launch("rumpy_residual_norm_fwd");
}

extern "C" int64_t rumpy_residual_norm_partial_floats(int64_t rows, int64_t group_rows, int32_t C, int32_t gate_mode) {
  if (rows <= 0 || C < 1 || C > RN_MAXC || (gate_mode == RN_GATE_GROUP && group_rows < 1)) return 0;
  const RnPlan plan = rn_plan(rows, group_rows, C, gate_mode);
  int64_t n = (int64_t)4 * plan.wgs;
  if (gate_mode == RN_GATE_GROUP) n += plan.direct ? rows : plan.wgs + (rows + group_rows - 1) / group_rows;
  return n * C;
}

extern "C" int rumpy_residual_norm_bwd(const rumpy_residual_norm_bwd_args* p, void* stream) {
  const char* bad = !p ? "no arguments" : rn_check(p->rows, p->group_rows, p->C, p->x_fmt, p->t_fmt, p->t, p->gate, p->gate_mode, p->post, p->pre);
  if (!bad && p->rows < 1) bad = "a backward pass has rows";
  if (!bad && (!p->x || !p->partial || (!p->dy && !p->dh))) bad = "a tensor is missing";
  if (!bad && (p->dh && p->pre == RN_NONE)) bad = "dh without a norm in front";
  if (!bad && ((p->post != RN_NONE || p->dh) && !p->stats)) bad = "the statistics of the forward pass are missing";
  if (!bad && (p->ldx < 0 || p->ldt < 0 || p->ldg < 0 || p->lddy < 0 || p->lddh < 0)) bad = "row strides are not negative";
  if (!bad && (!p->t && (p->dt || p->dgate || p->d_post_w || p->d_post_b))) bad = "a gradient of a branch that is not there";
  if (!bad && (p->gate_mode == RN_GATE_NONE && p->dgate)) bad = "a gradient of a gate that is not there";
  if (!bad && ((p->post == RN_NONE && (p->d_post_w || p->d_post_b)) || (!p->dh && (p->d_pre_w || p->d_pre_b)))) bad = "a gradient of a norm that is not there";
  const bool gate_rows = !bad && p->gate_mode == RN_GATE_GROUP && p->dgate;
  const int tiles = bad ? 0 : (p->C + 63) / 64;
  const int64_t items = 4 + (gate_rows ? p->rows / p->group_rows : 0);
  if (!bad && items * tiles > 0x7fffffff) bad = "too many gate rows";
  if (bad) { rumpy_set_error("rumpy_residual_norm_bwd: %s", bad); return RUMPY_E_ARG; }
  const RnPlan plan = rn_plan(p->rows, p->group_rows, p->C, p->gate_mode);
  hipStream_t s = (hipStream_t)stream;
  RN_BY_FORMAT(rn_launch_bwd, *p, plan, s);
  if (gate_rows || p->d_post_w || p->d_post_b || p->d_pre_w || p->d_pre_b)
    hipLaunchKernelGGL(residual_norm_reduce_kernel, dim3((unsigned)(items * tiles)), dim3(256), 0, s, *p, plan, tiles);
  return rumpy_check_launch("rumpy_residual_norm_bwd");
}
