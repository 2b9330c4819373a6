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
// Measured (MI355X, 5.2 TB/s for a large copy): 8192 x 4096 bf16 with a gate per element, forward 63 us = 5.3 TB/s, backward 100 us = 5.4 TB/s;
// 73728 x 64 bf16 with a gate per image 9.2 - 9.9 us = 4.0 TB/s and 18 us + 4 us of column sums (3.1 TB/s: the parts of a launch that are not
// the walk, for 5 steps of it); 4101 x 1001 fp32 + bf16 at odd strides 13 us = 3.8 TB/s, 19 + 6 us; one row of 4096 2.9 us.
#include "row_vec.hpp"
#include <type_traits>

constexpr int RN_GATE_NONE = 0, RN_GATE_GROUP = 1, RN_GATE_FULL = 2;
constexpr int RN_NONE = 0, RN_LAYER = 1, RN_RMS = 2;   // (RUMPY_FMT_*, gate modes and kinds are the header's)
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

// Where a lane's 8 channels lie.  The last piece of a row is moved back to end with the row, and lanes behind it repeat it: every access is one
// whole 16- or 32-byte access inside the row, with no branch around it.  What two lanes both hold they compute and store alike; in a row's sums
// the repeated elements count zero times (`m`, bits and not factors: an infinity is not made NaN).  Rows of up to 8 channels have one lane
// (TPR 1), with partial accesses under 8.
template <int TPR> struct RnLane {
  int at, n;             // first channel; channels of an access (TPR 1)
  uint32_t m[8];
  __device__ __forceinline__ explicit RnLane(int C) {
    const int col = ((int)threadIdx.x % TPR) * 8;
    at = TPR == 1 ? 0 : min(col, C - 8);
    n = TPR == 1 ? C : 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = (TPR == 1 ? i < C : i >= col - at) ? 0xffffffffu : 0u;
  }
  __device__ __forceinline__ float once(float v, int i) const { return __uint_as_float(__float_as_uint(v) & m[i]); }
  template <int FMT> __device__ __forceinline__ RowRaw<FMT> load(const void* base, size_t row_off) const {
    return load_piece<FMT>((const typename RowElem<FMT>::type*)base + row_off + at, TPR == 1 ? n : 8, 0.f);
  }
  template <int FMT> __device__ __forceinline__ void store(void* base, size_t row_off, const float (&v)[8]) const {
    store8<FMT>(base, row_off + at, TPR == 1 ? n : 8, v);
  }
  // fp32 parameters; NULL: the default
  __device__ __forceinline__ void params(const float* p, float dflt, float (&o)[8]) const {
    if (p) unpack_piece<RUMPY_FMT_F32>(load<RUMPY_FMT_F32>(p, 0), o);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = dflt;
    }
  }
};

// mean and 1 / sqrt(var + eps) of a row.  The variance is taken around the mean in a second sum (the row is in registers): no cancellation
// where the mean is large.  v_rsq_f32 is right to one unit in the last place for normal arguments (eps is one).
template <int TPR> __device__ __forceinline__ void row_stats(RowSum<TPR>& sum, const float (&v)[8], const RnLane<TPR>& lane, int kind, float inv_c, float eps,
                                                             float& mu, float& rs) {
  mu = 0.f;
  if (kind == RN_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += lane.once(v[i], i);
    mu = sum.one(s) * inv_c;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) { const float d = lane.once(v[i] - mu, i); q = fmaf(d, d, q); }
  rs = __builtin_amdgcn_rsqf(sum.one(q) * inv_c + eps);
}

// The grid holds what the chip runs at once and every workgroup walks over rows; a row's tensors are asked for before the row in front of it
// is computed, and unpacked behind that row's stores.  The counter that loads and stores share counts in order: where the number of stores in
// between is known, the wait for the loads leaves the stores in flight, so the usual calls (t, y and h; with or without statistics) are kernels of
// their own (MODE) and everything else is RN_ANY.  Rows behind the last one repeat it: they store the same values once more.
// (8192 x 4096: 101 us with a launch per 2 rows and parameters loaded one by one, 74 with the loads a row ahead, 63 with this order.)
constexpr int RN_ANY = 0, RN_EVAL = 1, RN_TRAIN = 2;
template <int XF, int TF, int TPR, int MODE> __global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR) residual_norm_fwd_kernel(rumpy_residual_norm_args a) {
  constexpr int WG = TPR <= 64 ? 256 : TPR, SUB = WG / TPR;
  __shared__ float red[2][2 * RowSum<TPR>::WAVES];
  RowSum<TPR> sum{red, 0};
  const RnLane<TPR> lane(a.C);
  const int sub = (int)threadIdx.x / TPR;
  const float inv_c = 1.f / (float)a.C;
  const uint32_t rows = (uint32_t)a.rows, step = gridDim.x * SUB;
  const bool has_t = MODE != RN_ANY || a.t, has_pre = MODE != RN_ANY || a.pre != RN_NONE, keep = MODE == RN_TRAIN || (MODE == RN_ANY && a.stats);
  uint32_t rb = blockIdx.x * SUB;
  // the gate row of the row that is asked for next, advanced without a division per row
  uint32_t grp = 0, rem = 0, grp_step = 0, rem_step = 0;
  const bool grouped = a.gate_mode == RN_GATE_GROUP, full = a.gate_mode == RN_GATE_FULL;
  if (grouped) {
    const uint32_t gr = (uint32_t)a.group_rows;
    grp = (rb + sub) / gr; rem = (rb + sub) % gr;
    grp_step = step / gr; rem_step = step % gr;
  }
  const uint32_t last_grp = grouped ? (rows - 1) / (uint32_t)a.group_rows : 0;
  RowRaw<XF> rx;
  RowRaw<TF> rt, rg;
  RowRaw<RUMPY_FMT_F32> rgate;
  auto ask = [&](uint32_t base) {
    const size_t r = min(base + sub, rows - 1);
    rx = lane.template load<XF>(a.x, r * a.ldx);
    if (has_t) rt = lane.template load<TF>(a.t, r * a.ldt);
    if (full) rg = lane.template load<TF>(a.gate, r * a.ldg);
    if (grouped) {
      rgate = lane.template load<RUMPY_FMT_F32>(a.gate, (size_t)min(grp, last_grp) * a.C);
      grp += grp_step; rem += rem_step;
      if (rem >= (uint32_t)a.group_rows) { rem -= (uint32_t)a.group_rows; ++grp; }
    }
  };
  float x[8], t[8], g[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { t[i] = 0.f; g[i] = 1.f; }
  auto take = [&]() {
    unpack_piece<XF>(rx, x);
    if (has_t) unpack_piece<TF>(rt, t);
    if (full) unpack_piece<TF>(rg, g);
    if (grouped) unpack_piece<RUMPY_FMT_F32>(rgate, g);
  };
  ask(rb);
  float wp[8], bp[8], w[8], b[8];
  lane.params(a.post_w, 1.f, wp);
  lane.params(a.post_b, 0.f, bp);
  lane.params(a.pre_w, 1.f, w);
  lane.params(a.pre_b, 0.f, b);
  take();
  while (true) {
    const size_t r = min(rb + sub, rows - 1);
    const bool more = rows - rb > step;
    ask(more ? rb + step : rb);
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (has_t) {
      if (a.post != RN_NONE) row_stats<TPR>(sum, t, lane, a.post, inv_c, a.eps, st.x, st.y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(a.scale * g[i], fmaf((t[i] - st.x) * st.y, wp[i], bp[i]), x[i]);
      lane.template store<XF>(a.y, r * a.C, x);
    }
    if (has_pre) {
      row_stats<TPR>(sum, x, lane, a.pre, inv_c, a.eps, st.z, st.w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf((x[i] - st.z) * st.w, w[i], b[i]);
      lane.template store<TF>(a.h, r * a.C, x);
    }
    if (keep) reinterpret_cast<float4*>(a.stats)[r] = st;
    if (!more) break;
    take();
    rb += step;
  }
}

// ---- backward ----
// Work of one launch: `wgs` workgroups of `rpw` contiguous rows each.  A gate row that serves a group of rows is summed over a workgroup's part
// of the group and stored as partial row (workgroup + group): over the walk of all (workgroup, group) pairs that number grows strictly.  Groups
// shorter than a workgroup's step store one partial row per row instead (groups of one row: the gradient itself).
struct RnPlan { int tpr, sub, wgs, rpw; bool direct; };
// As few lanes a row as hold it: with 8 at the least, 1048576 x 8 bf16 took 51 us forward and 102 backward, now 15 and 32; 524288 x 16 29 and 55, now 13 and 22
// (rows of 3 channels, in partial accesses, stay at 2.5 and 5 times their bytes).
static RnPlan rn_plan(int64_t rows, int64_t group_rows, int32_t C, int gate_mode) {
  RnPlan p;
  p.tpr = 1;
  while (p.tpr * 8 < C) p.tpr *= 2;
  p.sub = p.tpr <= 64 ? 256 / p.tpr : 1;
  const int64_t steps = (rows + p.sub - 1) / p.sub;
  // two waves of these registers fit a SIMD: 512 threads a CU.  At least two steps each, so that the partial rows stay fewer than the rows
  const int64_t most = p.tpr <= 64 ? 512 : p.tpr <= 512 ? 256 * (512 / p.tpr) : 256;
  int64_t wgs = (steps + 1) / 2;
  if (wgs > most) wgs = most;
  p.rpw = (int)((steps + wgs - 1) / wgs * p.sub);
  p.wgs = (int)((rows + p.rpw - 1) / p.rpw);
  p.direct = gate_mode == RN_GATE_GROUP && (group_rows < p.sub || group_rows == 1);
  return p;
}

// sum over the lanes of a wave that hold the same channels of different rows (every TPR-th lane), in each of them, without the LDS crossbar
template <int TPR> __device__ __forceinline__ float steps_sum(float v, int lane) {
  if constexpr (TPR == 1) return wave64_sum(v, lane);
  if constexpr (TPR == 2) v += dpp_quad2(v);                                             // lane ^ 2
  if constexpr (TPR <= 4) {
    const int i = __float_as_int(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(i, i, 0x124, 0xF, 0xF, false));      // row_ror 4: with the next step all four of a row's
  }
  if constexpr (TPR <= 8) {
    const int i = __float_as_int(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(i, i, 0x128, 0xF, 0xF, false));      // row_ror 8: lane ^ 8
  }
  if constexpr (TPR <= 16) v += lane_xor16(v, lane >> 4);
  if constexpr (TPR <= 32) v += lane_xor32(v, lane);
  return v;
}
// column sums of a workgroup: the rows of a step lie side by side in its waves
template <int TPR> __device__ __forceinline__ void flush_columns(const RnLane<TPR>& lane, float (&acc)[8], float* dst, float* lds) {
  if constexpr (TPR <= 64) {
    const int tid = threadIdx.x, l = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = steps_sum<TPR>(acc[i], l);
    __syncthreads();
    if (l < TPR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) lds[(wave * 8 + i) * TPR + l] = acc[i];
    }
    __syncthreads();
    if (tid < TPR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = (lds[i * TPR + l] + lds[(8 + i) * TPR + l]) + (lds[(16 + i) * TPR + l] + lds[(24 + i) * TPR + l]);
      lane.template store<RUMPY_FMT_F32>(dst, 0, acc);
    }
  } else {
    lane.template store<RUMPY_FMT_F32>(dst, 0, acc);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
}

// (8192 x 4096: 182 us with the loads a row ahead and every wait for all loads and stores, 100 with the order of the forward kernel.)
// MODE as in the forward kernel: RN_ALL = dy, dh, t, dx, dt (and no gate of t's shape), RN_ALL_FULL = those and a gate of t's shape with its gradient.
constexpr int RN_ALL = 1, RN_ALL_FULL = 2;
template <int XF, int TF, int TPR, int MODE> __global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR) residual_norm_bwd_kernel(rumpy_residual_norm_bwd_args a, RnPlan plan) {
  constexpr int WG = TPR <= 64 ? 256 : TPR, SUB = WG / TPR;
  // 1024 threads leave 128 registers each: the parameters' sums lie in LDS (each thread's own, 128 KB; 1024 x 8192 bf16:
  // 56 us with spills instead, 30), parameters come from the caches per row and nothing is asked for ahead
  constexpr bool HOLD = TPR <= 512;
  __shared__ float4 sums[HOLD ? 1 : 4 * 2 * TPR];
  auto add = [&](int which, const float (&v)[8]) {
    float4* p = sums + which * 2 * TPR + threadIdx.x;
    float4 lo = p[0], hi = p[TPR];
    lo.x += v[0]; lo.y += v[1]; lo.z += v[2]; lo.w += v[3];
    hi.x += v[4]; hi.y += v[5]; hi.z += v[6]; hi.w += v[7];
    p[0] = lo; p[TPR] = hi;
  };
  __shared__ float red[2][2 * RowSum<TPR>::WAVES];
  __shared__ float cols[TPR <= 64 ? 4 * TPR * 8 : 1];
  RowSum<TPR> sum{red, 0};
  const RnLane<TPR> lane(a.C);
  const int sub = (int)threadIdx.x / TPR;
  const float inv_c = 1.f / (float)a.C;
  const uint32_t rows = (uint32_t)a.rows, r0 = min(rows, blockIdx.x * (uint32_t)plan.rpw), r1 = min(rows, r0 + (uint32_t)plan.rpw);
  // partial: [4][wgs][C], then the gate's partial rows
  float* gpart = plan.direct && a.group_rows == 1 ? (float*)a.dgate : a.partial + (size_t)4 * plan.wgs * a.C;
  const bool has_t = MODE != RN_ANY || a.t, has_dy = MODE != RN_ANY || a.dy, has_dh = MODE != RN_ANY || a.dh;
  const bool full = MODE == RN_ALL_FULL || (MODE == RN_ANY && a.gate_mode == RN_GATE_FULL);
  const bool direct = MODE != RN_ALL_FULL && plan.direct, group_sums = MODE != RN_ALL_FULL && a.gate_mode == RN_GATE_GROUP && !plan.direct;

  RowRaw<XF> rx, rdy;
  RowRaw<TF> rt, rdh, rg;
  float4 rst = make_float4(0.f, 1.f, 0.f, 1.f), st;
  float x[8], t[8], d[8], e[8], g[8];
  auto ask = [&](size_t r) {
    rx = lane.template load<XF>(a.x, r * a.ldx);
    if (has_t) rt = lane.template load<TF>(a.t, r * a.ldt);
    if (has_dy) rdy = lane.template load<XF>(a.dy, r * a.lddy);
    if (has_dh) rdh = lane.template load<TF>(a.dh, r * a.lddh);
    if (full) rg = lane.template load<TF>(a.gate, r * a.ldg);
    if (MODE != RN_ANY || a.stats) rst = reinterpret_cast<const float4*>(a.stats)[r];
  };
  auto take = [&]() {
    unpack_piece<XF>(rx, x);
    if (has_t) unpack_piece<TF>(rt, t);
    if (has_dy) unpack_piece<XF>(rdy, d);
    if (has_dh) unpack_piece<TF>(rdh, e);
    if (full) unpack_piece<TF>(rg, g);
    st = rst;
  };
  float wp[8], bp[8], w[8];
  float aw[8], ab[8], awp[8], abp[8], ag[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { aw[i] = ab[i] = awp[i] = abp[i] = ag[i] = t[i] = d[i] = e[i] = 0.f; g[i] = 1.f; }
  if (HOLD) { lane.params(a.post_w, 1.f, wp); lane.params(a.post_b, 0.f, bp); lane.params(a.pre_w, 1.f, w); }
  else {
    for (int i = 0; i < 8; ++i) sums[i * TPR + threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // one step: SUB rows; those behind the segment repeat its last row, `live` takes them out of the column sums (TAIL steps alone have any)
  auto step = [&](size_t r, bool live, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    if (!HOLD) { lane.params(a.post_w, 1.f, wp); lane.params(a.post_b, 0.f, bp); }
    if (direct) unpack_piece<RUMPY_FMT_F32>(lane.template load<RUMPY_FMT_F32>(a.gate, (size_t)((uint32_t)r / (uint32_t)a.group_rows) * a.C), g);
    if (has_t) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t[i] = (t[i] - st.x) * st.y;                                              // that
        x[i] = fmaf(a.scale * g[i], fmaf(t[i], wp[i], bp[i]), x[i]);               // y, unrounded
      }
    }
    if (!has_dy) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = 0.f;
    }
    if (has_dh) {
      if (!HOLD) lane.params(a.pre_w, 1.f, w);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = (x[i] - st.z) * st.w;                                              // yhat
        const float ea = TAIL && !live ? 0.f : e[i];
        if (HOLD) { ab[i] += ea; aw[i] = fmaf(ea, x[i], aw[i]); }
        else { ab[i] = ea; aw[i] = ea * x[i]; }
        e[i] *= w[i];
        const float em = lane.once(e[i], i);
        s1 += em;
        s2 = fmaf(em, x[i], s2);
      }
      if (!HOLD) {
        if (a.d_pre_w) add(2, aw);
        if (a.d_pre_b) add(3, ab);
      }
      sum.two(s1, s2);
      s1 = a.pre == RN_LAYER ? s1 * inv_c : 0.f;
      s2 *= inv_c;
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = fmaf(st.w, (e[i] - s1) - x[i] * s2, d[i]);
    }
    if (MODE != RN_ANY || a.dx) lane.template store<XF>(a.dx, r * a.C, d);
    if (has_t) {
      if (!HOLD) { lane.params(a.post_w, 1.f, wp); lane.params(a.post_b, 0.f, bp); }
      float s1 = 0.f, s2 = 0.f;
      float gr[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float dd = a.scale * d[i];
        gr[i] = dd * fmaf(t[i], wp[i], bp[i]);
        const float dz = g[i] * dd;
        if (!HOLD) { ag[i] += gr[i]; abp[i] = dz; awp[i] = dz * t[i]; }
        else if (!TAIL || live) { ag[i] += gr[i]; abp[i] += dz; awp[i] = fmaf(dz, t[i], awp[i]); }
        d[i] = dz * wp[i];
        const float dm = lane.once(d[i], i);
        s1 += dm;
        s2 = fmaf(dm, t[i], s2);
      }
      if (!HOLD) {
        if (a.d_post_w) add(0, awp);
        if (a.d_post_b) add(1, abp);
      }
      if (MODE == RN_ALL_FULL || (full && a.dgate)) lane.template store<TF>(a.dgate, r * a.C, gr);
      else if (direct && a.dgate) lane.template store<RUMPY_FMT_F32>(gpart, r * a.C, gr);
      if (a.post != RN_NONE) {
        sum.two(s1, s2);
        s1 = a.post == RN_LAYER ? s1 * inv_c : 0.f;
        s2 *= inv_c;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = st.y * ((d[i] - s1) - t[i] * s2);
      }
      if (MODE != RN_ANY || a.dt) lane.template store<TF>(a.dt, r * a.C, d);
    }
  };
  for (uint32_t seg = r0; seg < r1;) {
    uint32_t end = r1;
    size_t group = 0;
    if (group_sums) {
      group = seg / (uint32_t)a.group_rows;
      end = (uint32_t)min((int64_t)r1, (int64_t)(group + 1) * a.group_rows);
      unpack_piece<RUMPY_FMT_F32>(lane.template load<RUMPY_FMT_F32>(a.gate, group * a.C), g);
    }
    const uint32_t last = end - 1;
    uint32_t rb = seg;
    if (HOLD) { ask(min(rb + sub, last)); take(); }
    for (; end - rb >= SUB && rb < end; rb += SUB) {
      if (HOLD) ask(min(rb + SUB + sub, last));
      else { ask(rb + sub); take(); }
      step(rb + sub, true, std::false_type());
      if (HOLD) take();
    }
    if (SUB > 1 && rb < end) {
      if (!HOLD) { ask(min(rb + sub, last)); take(); }
      step(min(rb + sub, last), rb + sub < end, std::true_type());
    }
    if (group_sums && a.dgate) flush_columns<TPR>(lane, ag, gpart + (blockIdx.x + group) * a.C, cols);
    seg = end;
  }
  if (!HOLD) {
    auto get = [&](int which, float (&v)[8]) {
      const float4 lo = sums[which * 2 * TPR + threadIdx.x], hi = sums[(which * 2 + 1) * TPR + threadIdx.x];
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    };
    get(0, awp); get(1, abp); get(2, aw); get(3, ab);
  }
  const size_t wc = (size_t)plan.wgs * a.C;
  float* mine = a.partial + (size_t)blockIdx.x * a.C;
  if (a.d_post_w) flush_columns<TPR>(lane, awp, mine, cols);
  if (a.d_post_b) flush_columns<TPR>(lane, abp, mine + wc, cols);
  if (a.d_pre_w) flush_columns<TPR>(lane, aw, mine + 2 * wc, cols);
  if (a.d_pre_b) flush_columns<TPR>(lane, ab, mine + 3 * wc, cols);
}

// out[c] = sum over consecutive partial rows: items 0..3 = the parameters (all workgroups), 4.. = the gate rows.  16 waves share a column's rows:
// with four a sum of 461 rows took 7 us of dependent loads.  Where there are many gate rows (`flat`), each of a few partial rows, a thread takes an element
// of one: a workgroup for 64 of them took 81 us for 32768 gate rows of 64 channels, 1650 for 700000 of 3; so 9 and 11.
constexpr int RN_SLICES = 16, RN_REDUCE_WG = 64 * RN_SLICES;
constexpr int64_t RN_FLAT_BLOCKS = 8192;      // their workgroups at most (a launch has fewer than 2^32 threads), which walk over the elements
// A thread's walk takes about 0.1 us a partial row, the workgroups of 64 columns 2.2 us a thousand: with more than 45 of them a partial row the threads win.  us,
// threads | workgroups:  65536 gate rows of 64 channels, 2 partial rows each: 18 | 148     4096 x 64, 31: 7.5 | 16.5     64 x 4096, 6: 5 | 17
// 1024 x 16, 127: 13.7 | 6.7     2048 x 8, 200: 19 | 14     8 x 4096, 33: 6.6 | 5.7     8 x 2048, 33: 8.2 | 4.9     2 x 8192, 130: 14 | 5.4
static bool rn_flat(const RnPlan& plan, int64_t groups, int64_t group_rows, int tiles) {
  const int64_t each = plan.direct ? group_rows : group_rows / plan.rpw + 2;
  return groups * tiles > 45 * each;
}
__device__ __forceinline__ const float* gate_partials(const rumpy_residual_norm_bwd_args& a, const RnPlan& plan, int64_t group, int64_t& count) {
  const int64_t first = group * a.group_rows, last = min(a.rows, first + a.group_rows) - 1;
  const float* src = a.partial + (size_t)4 * plan.wgs * a.C;
  if (plan.direct) { count = last - first + 1; return src + (size_t)first * a.C; }
  const int64_t w0 = first / plan.rpw, w1 = last / plan.rpw;
  count = w1 - w0 + 1;
  return src + (size_t)(w0 + group) * a.C;
}
__global__ void __launch_bounds__(RN_REDUCE_WG) residual_norm_reduce_kernel(rumpy_residual_norm_bwd_args a, RnPlan plan, int tiles, int64_t flat) {
  __shared__ float red[RN_SLICES][64];
  const size_t item = blockIdx.x / tiles;
  const float* src;
  float* dst;
  int64_t count;
  if (item >= 4 && flat) {
    const int64_t step = (int64_t)(gridDim.x - 4 * tiles) * RN_REDUCE_WG;
    for (int64_t e0 = (int64_t)(blockIdx.x - 4 * tiles) * RN_REDUCE_WG; e0 + threadIdx.x < flat; e0 += step) {
      const int64_t g0 = e0 / a.C;
      const uint32_t off = (uint32_t)(e0 - g0 * a.C) + threadIdx.x;
      src = gate_partials(a, plan, g0 + off / (uint32_t)a.C, count) + off % (uint32_t)a.C;
      float s = 0.f;
#pragma unroll 4
      for (int64_t i = 0; i < count; ++i) s += src[(size_t)i * a.C];
      ((float*)a.dgate)[e0 + threadIdx.x] = s;
    }
    return;
  }
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6, c = (blockIdx.x % tiles) * 64 + lane;
  if (item < 4) {
    dst = item == 0 ? a.d_post_w : item == 1 ? a.d_post_b : item == 2 ? a.d_pre_w : a.d_pre_b;
    src = a.partial + item * (size_t)plan.wgs * a.C;
    count = plan.wgs;
  } else {
    dst = (float*)a.dgate + (item - 4) * a.C;
    src = gate_partials(a, plan, (int64_t)item - 4, count);
  }
  if (!dst) return;                                            // (the whole workgroup)
  float s = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int64_t i = slice; i < count; i += RN_SLICES) s += src[(size_t)i * a.C + c];
  }
  red[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < a.C) {
#pragma unroll
    for (int i = 1; i < RN_SLICES; ++i) s += red[i][lane];
    dst[c] = s;
  }
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

// the usual calls have kernels of their own, from 9 channels on
template <int XF, int TF, int TPR> static void rn_launch_fwd_tpr(const rumpy_residual_norm_args& a, const dim3& grid, hipStream_t s) {
  const dim3 wg(TPR <= 64 ? 256 : TPR);
  if (TPR > 1 && a.t && a.pre != RN_NONE) {
    if (a.stats) hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, TPR, TPR == 1 ? RN_ANY : RN_TRAIN>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, TPR, TPR == 1 ? RN_ANY : RN_EVAL>), grid, wg, 0, s, a);
  } else {
    hipLaunchKernelGGL((residual_norm_fwd_kernel<XF, TF, TPR, RN_ANY>), grid, wg, 0, s, a);
  }
}
template <int XF, int TF, int TPR> static void rn_launch_bwd_tpr(const rumpy_residual_norm_bwd_args& a, const RnPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.wgs), wg(TPR <= 64 ? 256 : TPR);
  const bool all = TPR > 1 && a.dy && a.dh && a.t && a.dx && a.dt && a.stats;
  if (all && a.gate_mode != RN_GATE_FULL) hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, TPR, TPR == 1 ? RN_ANY : RN_ALL>), grid, wg, 0, s, a, p);
  else if (all && a.dgate) hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, TPR, TPR == 1 ? RN_ANY : RN_ALL_FULL>), grid, wg, 0, s, a, p);
  else hipLaunchKernelGGL((residual_norm_bwd_kernel<XF, TF, TPR, RN_ANY>), grid, wg, 0, s, a, p);
}
template <int XF, int TF> static void rn_launch_fwd(const rumpy_residual_norm_args& a, const RnPlan& p, hipStream_t s) {
  const int64_t steps = (a.rows + p.sub - 1) / p.sub;
  // four waves of these registers fit a SIMD: 1024 threads a CU
  const int64_t most = p.tpr <= 64 ? 1024 : 256 * 1024 / p.tpr;
  const dim3 grid((unsigned)(steps < most ? steps : most));
  switch (p.tpr) {
    case 1: return rn_launch_fwd_tpr<XF, TF, 1>(a, grid, s);
    case 2: return rn_launch_fwd_tpr<XF, TF, 2>(a, grid, s);
    case 4: return rn_launch_fwd_tpr<XF, TF, 4>(a, grid, s);
    case 8: return rn_launch_fwd_tpr<XF, TF, 8>(a, grid, s);
    case 16: return rn_launch_fwd_tpr<XF, TF, 16>(a, grid, s);
    case 32: return rn_launch_fwd_tpr<XF, TF, 32>(a, grid, s);
    case 64: return rn_launch_fwd_tpr<XF, TF, 64>(a, grid, s);
    case 128: return rn_launch_fwd_tpr<XF, TF, 128>(a, grid, s);
    case 256: return rn_launch_fwd_tpr<XF, TF, 256>(a, grid, s);
    case 512: return rn_launch_fwd_tpr<XF, TF, 512>(a, grid, s);
    default: return rn_launch_fwd_tpr<XF, TF, 1024>(a, grid, s);
  }
}
template <int XF, int TF> static void rn_launch_bwd(const rumpy_residual_norm_bwd_args& a, const RnPlan& p, hipStream_t s) {
  switch (p.tpr) {
    case 1: return rn_launch_bwd_tpr<XF, TF, 1>(a, p, s);
    case 2: return rn_launch_bwd_tpr<XF, TF, 2>(a, p, s);
    case 4: return rn_launch_bwd_tpr<XF, TF, 4>(a, p, s);
    case 8: return rn_launch_bwd_tpr<XF, TF, 8>(a, p, s);
    case 16: return rn_launch_bwd_tpr<XF, TF, 16>(a, p, s);
    case 32: return rn_launch_bwd_tpr<XF, TF, 32>(a, p, s);
    case 64: return rn_launch_bwd_tpr<XF, TF, 64>(a, p, s);
    case 128: return rn_launch_bwd_tpr<XF, TF, 128>(a, p, s);
    case 256: return rn_launch_bwd_tpr<XF, TF, 256>(a, p, s);
    case 512: return rn_launch_bwd_tpr<XF, TF, 512>(a, p, s);
    default: return rn_launch_bwd_tpr<XF, TF, 1024>(a, p, s);
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
  if (!bad && ((uintptr_t)p->stats & 15)) bad = "stats lies at a multiple of 16 bytes";
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
  if (gate_mode == RN_GATE_GROUP) n += plan.direct ? (group_rows == 1 ? 0 : rows) : plan.wgs + (rows + group_rows - 1) / group_rows;
  return n * C;
}

extern "C" int rumpy_residual_norm_bwd(const rumpy_residual_norm_bwd_args* p, void* stream) {
  const char* bad = !p ? "no arguments" : rn_check(p->rows, p->group_rows, p->C, p->x_fmt, p->t_fmt, p->t, p->gate, p->gate_mode, p->post, p->pre);
  if (!bad && p->rows < 1) bad = "a backward pass has rows";
  if (!bad && (!p->x || !p->partial || (!p->dy && !p->dh))) bad = "a tensor is missing";
  if (!bad && (p->dh && p->pre == RN_NONE)) bad = "dh without a norm in front";
  if (!bad && ((p->post != RN_NONE || p->dh) && !p->stats)) bad = "the statistics of the forward pass are missing";
  if (!bad && ((uintptr_t)p->stats & 15)) bad = "stats lies at a multiple of 16 bytes";
  if (!bad && (p->ldx < 0 || p->ldt < 0 || p->ldg < 0 || p->lddy < 0 || p->lddh < 0)) bad = "row strides are not negative";
  if (!bad && (!p->t && (p->dt || p->dgate || p->d_post_w || p->d_post_b))) bad = "a gradient of a branch that is not there";
  if (!bad && (p->gate_mode == RN_GATE_NONE && p->dgate)) bad = "a gradient of a gate that is not there";
  if (!bad && ((p->post == RN_NONE && (p->d_post_w || p->d_post_b)) || (!p->dh && (p->d_pre_w || p->d_pre_b)))) bad = "a gradient of a norm that is not there";
  const RnPlan plan = bad ? RnPlan{} : rn_plan(p->rows, p->group_rows, p->C, p->gate_mode);
  const bool gate_rows = !bad && p->gate_mode == RN_GATE_GROUP && p->dgate && !(plan.direct && p->group_rows == 1);
  const int tiles = bad ? 0 : (p->C + 63) / 64;
  const int64_t groups = gate_rows ? p->rows / p->group_rows : 0, flat = gate_rows && rn_flat(plan, groups, p->group_rows, tiles) ? groups * p->C : 0;
  const int64_t walk = (flat + RN_REDUCE_WG - 1) / RN_REDUCE_WG;
  const int64_t blocks = (flat ? 4 : 4 + groups) * tiles + (walk < RN_FLAT_BLOCKS ? walk : RN_FLAT_BLOCKS);
  if (bad) { rumpy_set_error("rumpy_residual_norm_bwd: %s", bad); return RUMPY_E_ARG; }
  hipStream_t s = (hipStream_t)stream;
  RN_BY_FORMAT(rn_launch_bwd, *p, plan, s);
  if (gate_rows || p->d_post_w || p->d_post_b || p->d_pre_w || p->d_pre_b)
    hipLaunchKernelGGL(residual_norm_reduce_kernel, dim3((unsigned)blocks), dim3(RN_REDUCE_WG), 0, s, *p, plan, tiles, flat);
  return rumpy_check_launch("rumpy_residual_norm_bwd");
}
