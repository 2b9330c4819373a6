// Distillation from a teacher's top logits: the selection of the teacher's k largest logits of every row, the loss of a student against them,
// and the loss's gradient.  With u = z / tau, q = softmax(u) over all V columns, p the teacher's distribution over the columns it lists (and,
// when `tail` is given, the rest of the columns as one more outcome of probability p_t):
//   l = tau^2 [ sum_i p_i (log p_i - log q_i) + p_t (log p_t - log q_t) ],   q_t = sum of q over the columns that are not listed
//   dl/dz_j = tau (q_j - p_j) listed ;  tau q_j (1 - p_t / q_t) not listed       (no tail: p_t = 0, sum p = 1)
// Rows are [V] fp32 / bf16 / fp16 of 8192 (the contrastive queue) to a few 100 000 columns.  Selection and loss read each row once (plus the
// selection's second look, from the caches), the gradient reads it once and writes it once: bound by memory, with one exponential per element
// and direction beside it.  The sum of exp runs over the row once with a running maximum per thread; q_t is summed directly over the columns
// that are not listed (a bit map of them lies in LDS): 1 - sum q_i would cancel where the listed columns hold nearly everything.
// All sums and exponentials are fp32; every reduction has a fixed order, so results are bitwise reproducible.
#include "row_vec.hpp"

constexpr int DS_MAXK = 256, DS_MAXV = 1 << 30;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float wave_max(float v, int lane) {
  v = fmaxf(v, dpp_quad1(v)); v = fmaxf(v, dpp_quad2(v)); v = fmaxf(v, dpp_half_mirror(v)); v = fmaxf(v, dpp_row_mirror(v));
  v = fmaxf(v, lane_xor16(v, lane >> 4));
  return fmaxf(v, lane_xor32(v, lane));
}
template <int WAVES> __device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave64_sum(v, threadIdx.x & 63);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) s += red[i];
  return s;
}
template <int WAVES> __device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v, threadIdx.x & 63);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) s = fmaxf(s, red[i]);
  return s;
}

// ================================================================================================================ selection
// order of the values as unsigned integers: -inf lowest, NaN highest, -0 = +0
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

constexpr int TL_WG = 512, TL_WAVES = TL_WG / 64, TL_CAP = 2048;

// fn(values, first column, count) over the row's pieces of CH elements, piece by piece over the threads; elements outside hold -inf
template <int FMT, int CH, typename Fn> __device__ __forceinline__ void for_pieces(const typename RowElem<FMT>::type* z, int V, Fn fn) {
  for (int64_t j = (int64_t)threadIdx.x * CH; j < V; j += TL_WG * CH) {
    float v[8];
    if constexpr (CH == 8) unpack_piece<FMT>(load_piece<FMT>(z + j, (int)min((int64_t)8, V - j), -INFINITY), v);
    else v[0] = elem_to_f32<FMT>(z[j]);
    fn(v, (int)j);
  }
}

// a bound that at least k of the row's elements reach: per wave the value that ceil(k / waves) of its lanes' maxima reach (a bitwise search on
// ballots), the smallest of them over the waves
template <int FMT, int CH> __device__ __forceinline__ float top_bound(const typename RowElem<FMT>::type* z, int V, int k, float* red) {
  float mx = -INFINITY;
  for_pieces<FMT, CH>(z, V, [&](const float (&v)[8], int) {
#pragma unroll
    for (int i = 0; i < CH; ++i) mx = fmaxf(mx, v[i]);            // (NaN is passed over here; the second look meets it)
  });
  const uint32_t key = order_key(mx);
  const int want = (k + TL_WAVES - 1) / TL_WAVES;
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t trial = t | (1u << bit);
    if (__popcll(__ballot(key >= trial)) >= want) t = trial;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = key_value(t);
  __syncthreads();
  float T = red[0];
#pragma unroll
  for (int i = 1; i < TL_WAVES; ++i) T = fminf(T, red[i]);
  return T;
}
// the second look: collects what reaches T; returns this thread's sum of exp2((z - T) c) over the rest
template <int FMT, int CH> __device__ __forceinline__ float collect(const typename RowElem<FMT>::type* z, int V, float T, float c, uint64_t* cand, uint32_t* found) {
  float sum = 0.f;
  const float m = T * c;
  for_pieces<FMT, CH>(z, V, [&](const float (&v)[8], int j) {
    float s = 0.f, top = -INFINITY;
#pragma unroll
    for (int i = 0; i < CH; ++i) { s += __builtin_amdgcn_exp2f(fmaf(v[i], c, -m)); top = fmaxf(top, v[i]); }
    if (top >= T) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (v[i] >= T) {
          const uint32_t at = atomicAdd(found, 1u);
          if (at < TL_CAP) cand[at] = ((uint64_t)order_key(v[i]) << 32) | (uint32_t)~(uint32_t)(j + i);
        } else {
          s += __builtin_amdgcn_exp2f(fmaf(v[i], c, -m));
        }
      }
    }
    sum += s;
  });
  return sum;
}
// log sum exp(z / tau) over the elements whose (key, ~index) pair lies below `kth`, by their maximum; every thread gets it
template <int FMT> __device__ __forceinline__ float rest_below(const typename RowElem<FMT>::type* z, int V, uint64_t kth, float c, float inv_tau, float* red) {
  float rmx = -INFINITY, bad = 0.f;
  for (int64_t j = threadIdx.x; j < V; j += TL_WG) {
    const float v = elem_to_f32<FMT>(z[j]);
    if ((((uint64_t)order_key(v) << 32) | (uint32_t)~(uint32_t)j) < kth) { rmx = fmaxf(rmx, v); if (v != v) bad = 1.f; }
  }
  rmx = block_max<TL_WAVES>(rmx, red);
  if (block_max<TL_WAVES>(bad, red) > 0.f) return __uint_as_float(0x7fc00000u);
  if (!(fabsf(rmx) < INFINITY)) return rmx;
  float s = 0.f;
  for (int64_t j = threadIdx.x; j < V; j += TL_WG) {
    const float v = elem_to_f32<FMT>(z[j]);
    if ((((uint64_t)order_key(v) << 32) | (uint32_t)~(uint32_t)j) < kth) s += __builtin_amdgcn_exp2f((v - rmx) * c);
  }
  s = block_sum<TL_WAVES>(s, red);
  return fmaf(rmx, inv_tau, __builtin_amdgcn_logf(s) * LN2);
}

// One workgroup per row, two looks at it: the bound, then the few elements that reach it (a few times k) and the sum of exp over all others.
// A candidate's place is the number of candidates in front of it (larger value, or equal and lower index).  Rows whose bound collects too
// much or is not finite (fewer than about k finite elements), or that hold NaN, take the exact way: the k-th largest (value, index) pair by an
// 8-bit radix search over the row, which needs no assumption about the values.
template <int FMT> __global__ void __launch_bounds__(TL_WG) top_logits_kernel(rumpy_top_logits_args a) {
  typedef typename RowElem<FMT>::type E;
  __shared__ float red[TL_WAVES];
  __shared__ uint64_t cand[TL_CAP];
  __shared__ float after[TL_CAP];              // the candidates that are not chosen, by place: cand's own order is the atomics'
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found, need_s;
  __shared__ uint64_t prefix_s, kth_s, next_s;
  const int tid = threadIdx.x, V = a.V, k = a.k;
  const float c = a.inv_tau * LOG2E;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const E* z = reinterpret_cast<const E*>(a.logits) + (size_t)row * a.ld;
    uint32_t n = 0;
    float T = 0.f, sum = 0.f;
    bool exact_way = false;
    if (tid == 0) { found = 0; next_s = 0; }
    if (V <= TL_WG) {                                       // a row of one element per thread: all of them are candidates
      if (tid < V) cand[tid] = ((uint64_t)order_key(elem_to_f32<FMT>(z[tid])) << 32) | (uint32_t)~(uint32_t)tid;
      n = (uint32_t)V;
      __syncthreads();
    } else {
      // single elements instead of pieces where pieces would leave threads (whole waves, then) without any
      const bool pieces = V >= TL_WG * 8;
      T = pieces ? top_bound<FMT, 8>(z, V, k, red) : top_bound<FMT, 1>(z, V, k, red);
      exact_way = !(fabsf(T * c) < INFINITY) || !(fabsf(T) < INFINITY);
      if (!exact_way) {
        sum = pieces ? collect<FMT, 8>(z, V, T, c, cand, &found) : collect<FMT, 1>(z, V, T, c, cand, &found);
        sum = block_sum<TL_WAVES>(sum, red);
        n = found;
        exact_way = n > TL_CAP || sum != sum;
      }
    }
    if (exact_way) {
      // (key << 32 | ~index), 8 bits at a time from the top
      if (tid == 0) { prefix_s = 0; need_s = (uint32_t)k; }
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += TL_WG) hist[i] = 0;
        __syncthreads();
        const uint64_t prefix = prefix_s, mask = shift == 56 ? 0ull : ~0ull << (shift + 8);
        const int64_t rounds = ((int64_t)V + TL_WG - 1) / TL_WG;
        for (int64_t i = 0; i < rounds; ++i) {                   // (whole waves: the ballots below need every lane)
          const int64_t j = i * TL_WG + tid;
          bool in = j < V;
          uint64_t kk = 0;
          if (in) { kk = ((uint64_t)order_key(elem_to_f32<FMT>(z[j])) << 32) | (uint32_t)~(uint32_t)j; in = (kk & mask) == prefix; }
          const uint32_t bin = (uint32_t)(kk >> shift) & 255u;
          uint64_t left = __ballot(in);
          while (left) {                                       // one LDS add per distinct digit of the wave
            const int first = __ffsll((unsigned long long)left) - 1;
            const uint32_t b = __shfl(bin, first);
            const uint64_t same = __ballot(in && bin == b) & left;
            if ((tid & 63) == first) atomicAdd(&hist[b], (uint32_t)__popcll(same));
            left &= ~same;
          }
        }
        __syncthreads();
        if (tid == 0) {
          uint32_t need = need_s, b = 255;
          while (b > 0 && hist[b] < need) { need -= hist[b]; --b; }
          need_s = need;
          prefix_s = prefix | ((uint64_t)b << shift);
        }
        __syncthreads();
      }
      const uint64_t kth = prefix_s;                            // exactly k pairs are >= kth
      if (tid == 0) found = 0;
      __syncthreads();
      for (int64_t j = tid; j < V; j += TL_WG) {
        const uint64_t kk = ((uint64_t)order_key(elem_to_f32<FMT>(z[j])) << 32) | (uint32_t)~(uint32_t)j;
        if (kk >= kth) { const uint32_t at = atomicAdd(&found, 1u); if (at < TL_CAP) cand[at] = kk; }
      }
      n = (uint32_t)k;
      __syncthreads();
    }
    for (uint32_t i = tid; i < n; i += TL_WG) {
      const uint64_t mine = cand[i];
      uint32_t rank = 0;
      for (uint32_t o = 0; o < n; ++o) rank += cand[o] > mine;
      if (rank < (uint32_t)k) {
        const uint32_t idx = ~(uint32_t)mine;
        reinterpret_cast<E*>(a.values)[(size_t)row * k + rank] = z[idx];
        reinterpret_cast<int64_t*>(a.indices)[(size_t)row * k + rank] = idx;
        if (rank == (uint32_t)k - 1) kth_s = mine;
      } else {
        after[rank] = key_value((uint32_t)(mine >> 32));
        if (rank == (uint32_t)k) next_s = mine;
      }
    }
    __syncthreads();
    float tail;
    if (next_s == 0 && n < (uint32_t)V && (exact_way || sum < 1e-20f)) {
      // nothing collected beyond the top, and the others lie so far under the bound that their sum has no digits left (or was not made)
      tail = rest_below<FMT>(z, V, kth_s, c, a.inv_tau, red);
    } else {
      const float next = next_s ? key_value((uint32_t)(next_s >> 32)) : T;
      if (n == (uint32_t)V && next_s == 0) tail = -INFINITY;      // k = V: nothing is left
      else if (!(fabsf(next) < INFINITY)) tail = next;
      else {
        // relative to the largest that was not chosen: the other candidates, and the sum under the bound with T's distance from it
        float s = 0.f;
        for (uint32_t i = k + tid; i < n; i += TL_WG) s += __builtin_amdgcn_exp2f((after[i] - next) * c);
        s = block_sum<TL_WAVES>(s, red) + (sum > 0.f ? sum * __builtin_amdgcn_exp2f((T - next) * c) : 0.f);
        tail = fmaf(next, a.inv_tau, __builtin_amdgcn_logf(s) * LN2);
      }
    }
    if (tid == 0) a.tail[row] = tail;
    __syncthreads();
  }
}

extern "C" int rumpy_top_logits(const rumpy_top_logits_args* p, void* stream) {
  const char* bad = !p ? "no arguments" : nullptr;
  if (!bad && (p->fmt != RUMPY_FMT_F32 && p->fmt != RUMPY_FMT_BF16 && p->fmt != RUMPY_FMT_F16)) bad = "fp32, bf16 or fp16 logits";
  if (!bad && (p->rows < 0 || p->V < 1 || p->V > DS_MAXV || p->ld < 0)) bad = "rows of 1 .. 2^30 logits";
  if (!bad && (p->k < 1 || p->k > DS_MAXK || p->k > p->V)) bad = "1 .. 256 top logits, no more than the row has";
  if (!bad && !(p->inv_tau > 0.f && p->inv_tau < INFINITY)) bad = "a temperature above zero";
  if (!bad && p->rows && (!p->logits || !p->values || !p->indices || !p->tail)) bad = "a tensor is missing";
  if (bad) { rumpy_set_error("rumpy_top_logits: %s", bad); return RUMPY_E_ARG; }
  if (p->rows == 0) return RUMPY_OK;
  const dim3 grid((unsigned)(p->rows < 65536 ? p->rows : 65536));
  hipStream_t s = (hipStream_t)stream;
  if (p->fmt == RUMPY_FMT_F32) hipLaunchKernelGGL((top_logits_kernel<RUMPY_FMT_F32>), grid, dim3(TL_WG), 0, s, *p);
  else if (p->fmt == RUMPY_FMT_BF16) hipLaunchKernelGGL((top_logits_kernel<RUMPY_FMT_BF16>), grid, dim3(TL_WG), 0, s, *p);
  else hipLaunchKernelGGL((top_logits_kernel<RUMPY_FMT_F16>), grid, dim3(TL_WG), 0, s, *p);
  return rumpy_check_launch("rumpy_top_logits");
}

// ================================================================================================================ loss and gradient
constexpr int DS_WG = 512, DS_WAVES = DS_WG / 64;
constexpr int DS_STATE = 8;      // per row: reference and coefficient of the streamed columns, maximum and log sum of all, the teacher's log sum, dead, the teacher's maximum

// exp((v - m) / tau) with c = log2(e) / tau.  One fused multiply-add per element needs m c finite: a type's lowest value (a mask) overflows
// there, and takes the difference first.  fl(m c) is off m c by a rounding, ds_off says how much (in powers of two).
__device__ __forceinline__ float ds_exp(float v, float m, float c, float mc) {
  return __builtin_amdgcn_exp2f(fabsf(mc) < INFINITY ? fmaf(v, c, -mc) : (v - m) * c);
}
__device__ __forceinline__ float ds_off(float m, float c) { const float mc = m * c; return fabsf(mc) < INFINITY ? fmaf(m, c, -mc) : 0.f; }
// the factor from a sum relative to m to one relative to M >= m.  Where a product overflows, different values are so far apart that it is 0.
__device__ __forceinline__ float ds_rescale(float m, float M, float c) {
  if (m == M) return 1.f;
  const float d = m * c - M * c;
  return m == -INFINITY || d != d ? 0.f : __builtin_amdgcn_exp2f(d);
}

struct DsPlan { int splits, seg; };
// rows are cut when there are too few of them to fill the chip; a piece's bit map of listed columns has to fit LDS (2^18 columns: 32 KB)
static DsPlan ds_plan(int64_t rows, int32_t V) {
  DsPlan p;
  int64_t s = rows > 0 ? (512 + rows - 1) / rows : 1;
  const int64_t most = (V + 8191) / 8192, least = ((int64_t)V + (1 << 18) - 1) >> 18;
  if (s > most) s = most;
  if (s > 256) s = 256;
  if (s < least) s = least;
  p.seg = (int)((((int64_t)V + s - 1) / s + 4095) / 4096 * 4096);
  p.splits = (int)(((int64_t)V + p.seg - 1) / p.seg);
  return p;
}

__device__ __forceinline__ int64_t ds_index(const rumpy_distill_args& a, int64_t row, int i) {
  const size_t at = (size_t)row * a.k + i;
  return a.index64 ? reinterpret_cast<const int64_t*>(a.top_indices)[at] : (int64_t)reinterpret_cast<const int32_t*>(a.top_indices)[at];
}
__device__ __forceinline__ float ds_value(const rumpy_distill_args& a, int64_t row, int i) {
  const size_t at = (size_t)row * a.k + i;
  return a.value_fmt == RUMPY_FMT_F32 ? load_elem<RUMPY_FMT_F32>(a.top_values, at)
       : a.value_fmt == RUMPY_FMT_F16 ? load_elem<RUMPY_FMT_F16>(a.top_values, at) : load_elem<RUMPY_FMT_BF16>(a.top_values, at);
}

// what the teacher lists of a row, in LDS.  idx -1 = an entry that is not used (negative index); -2 = outside the row (the row becomes NaN).
// first[i]: no earlier entry names the same column
struct DsListed { int idx[DS_MAXK]; float v[DS_MAXK]; float z[DS_MAXK]; uint8_t first[DS_MAXK]; };
template <int FMT> __device__ __forceinline__ void ds_load_listed(const rumpy_distill_args& a, int64_t row, const typename RowElem<FMT>::type* z, DsListed& l) {
  const int tid = threadIdx.x;
  if (tid < a.k) {
    const int64_t i = ds_index(a, row, tid);
    const bool inside = i >= 0 && i < a.V;
    l.idx[tid] = i < 0 ? -1 : inside ? (int)i : -2;
    l.v[tid] = ds_value(a, row, tid);
    l.z[tid] = inside ? elem_to_f32<FMT>(z[i]) : 0.f;
  }
  __syncthreads();
  if (tid < a.k) {
    bool f = true;
    const int mine = l.idx[tid];
    for (int o = 0; o < a.k; ++o) f &= !(o < tid && l.idx[o] == mine);
    l.first[tid] = f;
  }
}

// one wave: the row's loss and what its gradient needs, from the sum over the streamed columns (all of them, or the unlisted ones when the
// rest is an outcome): s = sum exp2(z c - fl(m c)).
__device__ __forceinline__ void ds_finish(const rumpy_distill_args& a, int64_t row, const DsListed& l, float m, float s, int lane) {
  const float inv_tau = a.inv_tau, c = inv_tau * LOG2E;
  const bool rest = a.tail != nullptr;
  const float w = a.row_weight ? a.row_weight[row] : 1.f;
  float vm = -INFINITY, zm = -INFINITY;
  bool odd = false, outside = false;
  for (int i = lane; i < a.k; i += 64) {
    if (l.idx[i] == -1) continue;
    outside |= l.idx[i] == -2;
    odd |= l.v[i] != l.v[i];
    vm = fmaxf(vm, l.v[i]);
    zm = fmaxf(zm, l.z[i]);
  }
  vm = wave_max(vm, lane);
  zm = wave_max(zm, lane);
  const float tl = rest ? a.tail[row] : -INFINITY;
  const bool nan = __ballot(odd || outside) != 0ull || tl != tl;
  float* st = a.state + row * DS_STATE;
  if (!nan && vm == -INFINITY && tl == -INFINITY) {            // the teacher says nothing about this row
    if (lane == 0) { a.row_loss[row] = 0.f; st[0] = st[1] = st[2] = st[3] = st[4] = 0.f; st[5] = 1.f; }
    return;
  }
  // the teacher's logarithms relative to its largest logit, so that far from zero no digits are lost: lp = (v - vm) / tau - up - ln_p
  if (vm == -INFINITY) vm = 0.f;
  const float tr = fmaf(-vm, inv_tau, tl), up = fmaxf(0.f, tr);
  const float M = rest ? fmaxf(m, zm) : m, Mc = M * c;
  float p_sum = 0.f, sl = 0.f;
  for (int i = lane; i < a.k; i += 64) {
    if (l.idx[i] < 0) continue;
    p_sum += __builtin_amdgcn_exp2f(((l.v[i] - vm) * inv_tau - up) * LOG2E);
    if (rest && l.first[i]) sl += ds_exp(l.z[i], M, c, Mc);
  }
  p_sum = wave64_sum(p_sum, lane) + (rest ? __builtin_amdgcn_exp2f((tr - up) * LOG2E) : 0.f);
  const float ln_p = __builtin_amdgcn_logf(p_sum) * LN2;
  float S = s;
  if (rest) S = wave64_sum(sl, lane) + (m == -INFINITY ? 0.f : s * ds_rescale(m, M, c));
  const float ln_s = (__builtin_amdgcn_logf(S) - ds_off(M, c)) * LN2;
  float loss = 0.f;
  for (int i = lane; i < a.k; i += 64) {
    if (l.idx[i] < 0) continue;
    const float lp = (l.v[i] - vm) * inv_tau - up - ln_p, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    if (p != 0.f) loss += p * (lp - ((l.z[i] - M) * inv_tau - ln_s));
  }
  loss = wave64_sum(loss, lane);
  float coef = 1.f / S;
  if (rest) {
    const float lpt = tr - up - ln_p, pt = __builtin_amdgcn_exp2f(lpt * LOG2E);
    const float lqt = m == -INFINITY ? -INFINITY : (m - M) * inv_tau + (__builtin_amdgcn_logf(s) - ds_off(m, c)) * LN2 - ln_s;
    const float qt = __builtin_amdgcn_exp2f(lqt * LOG2E);
    if (pt != 0.f) loss += pt * (lpt - lqt);
    coef = m == -INFINITY ? 0.f : (qt - pt) / s;
  }
  if (nan) loss = coef = __uint_as_float(0x7fc00000u);
  if (lane == 0) {
    a.row_loss[row] = w == 0.f ? 0.f : w * loss * a.tau * a.tau;
    st[0] = m == -INFINITY ? 0.f : m;
    st[1] = coef;
    st[2] = M;
    st[3] = nan ? coef : ln_s;
    st[4] = up + ln_p;
    st[5] = w == 0.f ? 1.f : 0.f;
    st[6] = vm;
  }
}

// One workgroup per piece of a row.  REST: the listed columns are left out of the sum (bit map in LDS).
template <int FMT, bool REST> __global__ void __launch_bounds__(DS_WG) distill_fwd_kernel(rumpy_distill_args a, DsPlan plan) {
  typedef typename RowElem<FMT>::type E;
  extern __shared__ uint32_t bits[];
  __shared__ float red[DS_WAVES];
  __shared__ DsListed l;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / plan.splits;
  const int piece = blockIdx.x % plan.splits;
  const E* z = reinterpret_cast<const E*>(a.logits) + (size_t)row * a.ld;
  if (a.row_weight && a.row_weight[row] == 0.f) {               // a row that does not count is not looked at
    if (plan.splits == 1 && tid == 0) { a.row_loss[row] = 0.f; a.state[row * DS_STATE + 5] = 1.f; }
    return;
  }
  const int64_t j0 = (int64_t)piece * plan.seg, j1 = min((int64_t)a.V, j0 + plan.seg);
  if (plan.splits == 1) ds_load_listed<FMT>(a, row, z, l);
  if constexpr (REST) {
    const int words = (int)((j1 - j0 + 31) / 32);
    for (int i = tid; i < words; i += DS_WG) bits[i] = 0;
    __syncthreads();
    if (tid < a.k) {
      const int64_t i = ds_index(a, row, tid);
      if (i >= j0 && i < j1) atomicOr(&bits[(i - j0) >> 5], 1u << ((i - j0) & 31));
    }
    __syncthreads();
  }
  const float c = a.inv_tau * LOG2E;
  float m = -INFINITY, s = 0.f, mc = 0.f;
  for (int64_t j = j0 + tid * 8; j < j1; j += DS_WG * 8) {
    float v[8];
    unpack_piece<FMT>(load_piece<FMT>(z + j, (int)min((int64_t)8, j1 - j), -INFINITY), v);
    if constexpr (REST) {
      const uint32_t here = reinterpret_cast<const uint8_t*>(bits)[(j - j0) >> 3];
      if (here) {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (here >> i & 1u) v[i] = -INFINITY;
      }
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, v[i]);
    if (top > m) {
      s *= ds_rescale(m, top, c);
      m = top;
      mc = top * c;
    }
    if (fabsf(mc) < INFINITY) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s += __builtin_amdgcn_exp2f(fmaf(v[i], c, -mc));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) s += __builtin_amdgcn_exp2f((v[i] - m) * c);
    }
  }
  const float M = block_max<DS_WAVES>(m, red);
  s = block_sum<DS_WAVES>(m == -INFINITY ? s : s * ds_rescale(m, M, c), red);
  if (plan.splits > 1) {
    if (tid == 0) { a.partial[blockIdx.x * (size_t)2] = M; a.partial[blockIdx.x * (size_t)2 + 1] = s; }
    return;
  }
  if (tid < 64) ds_finish(a, row, l, M, s, tid);
}

// rows that were cut: their pieces' sums, then the row
template <int FMT> __global__ void __launch_bounds__(DS_WG) distill_join_kernel(rumpy_distill_args a, DsPlan plan) {
  typedef typename RowElem<FMT>::type E;
  __shared__ float red[DS_WAVES];
  __shared__ DsListed l;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  if (a.row_weight && a.row_weight[row] == 0.f) {
    if (tid == 0) { a.row_loss[row] = 0.f; a.state[row * DS_STATE + 5] = 1.f; }
    return;
  }
  ds_load_listed<FMT>(a, row, reinterpret_cast<const E*>(a.logits) + (size_t)row * a.ld, l);
  const float c = a.inv_tau * LOG2E;
  const float* part = a.partial + (size_t)row * plan.splits * 2;
  float m = -INFINITY;
  for (int i = tid; i < plan.splits; i += DS_WG) m = fmaxf(m, part[2 * i]);
  const float M = block_max<DS_WAVES>(m, red);
  float s = 0.f;
  for (int i = tid; i < plan.splits; i += DS_WG) {
    const float mi = part[2 * i];
    s += mi == -INFINITY ? part[2 * i + 1] : part[2 * i + 1] * ds_rescale(mi, M, c);
  }
  s = block_sum<DS_WAVES>(s, red);
  if (tid < 64) ds_finish(a, row, l, M, s, tid);
}

// loss = sum of the rows' (weighted) losses, over the sum of the weights for the mean; a sum of weights of zero gives 0
__global__ void __launch_bounds__(DS_WG) distill_total_kernel(rumpy_distill_args a) {
  __shared__ float red[DS_WAVES];
  float s = 0.f, w = 0.f;
  for (int64_t r = threadIdx.x; r < a.rows; r += DS_WG) { s += a.row_loss[r]; w += a.row_weight ? a.row_weight[r] : 1.f; }
  s = block_sum<DS_WAVES>(s, red);
  w = block_sum<DS_WAVES>(w, red);
  if (threadIdx.x == 0) {
    const float f = !a.mean ? 1.f : w == 0.f ? 0.f : 1.f / w;
    *a.factor = f;
    *a.loss = f == 0.f ? 0.f : s * f;
  }
}

template <int FMT> __global__ void __launch_bounds__(DS_WG) distill_bwd_kernel(rumpy_distill_args a, DsPlan plan) {
  typedef typename RowElem<FMT>::type E;
  __shared__ int idx[DS_MAXK];
  __shared__ float p[DS_MAXK];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / plan.splits;
  const int piece = blockIdx.x % plan.splits;
  const E* z = reinterpret_cast<const E*>(a.logits) + (size_t)row * a.ld;
  const int64_t j0 = (int64_t)piece * plan.seg, j1 = min((int64_t)a.V, j0 + plan.seg);
  const float* st = a.state + row * DS_STATE;
  const size_t out = (size_t)row * a.V;
  if (st[5] != 0.f) {
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t j = j0 + tid * 8; j < j1; j += DS_WG * 8) store8<FMT>(a.dlogits, out + j, (int)min((int64_t)8, j1 - j), zero);
    return;
  }
  const float c = a.inv_tau * LOG2E;
  float g = (a.loss ? *a.gout * *a.factor : a.gout[row]) * a.tau;
  if (a.row_weight) g *= a.row_weight[row];
  const float m = st[0], mc = m * c, coef = g * st[1];
  const bool fused = fabsf(mc) < INFINITY;
  if (tid < a.k) {
    const int64_t i = ds_index(a, row, tid);
    idx[tid] = i >= j0 && i < j1 ? (int)i : -1;
    p[tid] = i < 0 ? 0.f : __builtin_amdgcn_exp2f(((ds_value(a, row, tid) - st[6]) * a.inv_tau - st[4]) * LOG2E);
  }
  for (int64_t j = j0 + tid * 8; j < j1; j += DS_WG * 8) {
    const int n = (int)min((int64_t)8, j1 - j);
    float v[8];
    unpack_piece<FMT>(load_piece<FMT>(z + j, n, 0.f), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = coef * __builtin_amdgcn_exp2f(fused ? fmaf(v[i], c, -mc) : (v[i] - m) * c);
    store8<FMT>(a.dlogits, out + j, n, v);
  }
  __syncthreads();          // the listed columns are written over (same workgroup, behind the barrier); a column listed twice takes both shares
  if (tid < a.k && idx[tid] >= 0) {
    float share = 0.f;
    for (int o = 0; o < a.k; ++o) share += idx[o] == idx[tid] ? p[o] : 0.f;
    const float q = __builtin_amdgcn_exp2f(((elem_to_f32<FMT>(z[idx[tid]]) - st[2]) * a.inv_tau - st[3]) * LOG2E);
    reinterpret_cast<E*>(a.dlogits)[out + idx[tid]] = f32_to_elem<FMT>(g * (q - share));
  }
}

static bool ds_fmt(int f) { return f == RUMPY_FMT_F32 || f == RUMPY_FMT_BF16 || f == RUMPY_FMT_F16; }
static const char* ds_check(const rumpy_distill_args* p) {
  if (!p) return "no arguments";
  if (!ds_fmt(p->fmt) || !ds_fmt(p->value_fmt)) return "fp32, bf16 or fp16 logits and top logits";
  if (p->rows < 0 || p->V < 1 || p->V > DS_MAXV || p->ld < 0) return "rows of 1 .. 2^30 logits";
  if (p->k < 1 || p->k > DS_MAXK) return "1 .. 256 top logits a row";
  if (!(p->tau > 0.f && p->tau < INFINITY && p->inv_tau > 0.f && p->inv_tau < INFINITY)) return "a temperature above zero";
  if (p->rows && (!p->logits || !p->top_values || !p->top_indices || !p->row_loss || !p->state)) return "a tensor is missing";
  if (p->loss && !p->factor) return "the reduction's factor is missing";
  const DsPlan plan = ds_plan(p->rows, p->V);
  if (p->rows * plan.splits > 0x7fffffff) return "too many rows";
  if (plan.splits > 1 && !p->partial) return "rows of this length and number are cut and need `partial` (rumpy_distill_partial_floats)";
  return nullptr;
}
extern "C" int64_t rumpy_distill_partial_floats(int64_t rows, int32_t V) {
  if (rows <= 0 || V < 1 || V > DS_MAXV) return 0;
  const DsPlan plan = ds_plan(rows, V);
  return plan.splits > 1 ? rows * plan.splits * 2 : 0;
}

template <int FMT> static void ds_launch_fwd(const rumpy_distill_args& a, const DsPlan& plan, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * plan.splits));
  const size_t lds = a.tail ? ((size_t)(plan.splits == 1 ? a.V : plan.seg) + 31) / 32 * 4 : 0;
  if (a.tail) hipLaunchKernelGGL((distill_fwd_kernel<FMT, true>), grid, dim3(DS_WG), lds, s, a, plan);
  else hipLaunchKernelGGL((distill_fwd_kernel<FMT, false>), grid, dim3(DS_WG), 0, s, a, plan);
  if (plan.splits > 1) hipLaunchKernelGGL((distill_join_kernel<FMT>), dim3((unsigned)a.rows), dim3(DS_WG), 0, s, a, plan);
}
extern "C" int rumpy_distill_fwd(const rumpy_distill_args* p, void* stream) {
  const char* bad = ds_check(p);
  if (bad) { rumpy_set_error("rumpy_distill_fwd: %s", bad); return RUMPY_E_ARG; }
  hipStream_t s = (hipStream_t)stream;
  if (p->rows) {
    const DsPlan plan = ds_plan(p->rows, p->V);
    if (p->fmt == RUMPY_FMT_F32) ds_launch_fwd<RUMPY_FMT_F32>(*p, plan, s);
    else if (p->fmt == RUMPY_FMT_BF16) ds_launch_fwd<RUMPY_FMT_BF16>(*p, plan, s);
    else ds_launch_fwd<RUMPY_FMT_F16>(*p, plan, s);
  }
  if (p->loss) hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(DS_WG), 0, s, *p);
  return rumpy_check_launch("rumpy_distill_fwd");
}
extern "C" int rumpy_distill_bwd(const rumpy_distill_args* p, void* stream) {
  const char* bad = ds_check(p);
  if (!bad && p->rows && (!p->dlogits || !p->gout)) bad = "a tensor is missing";
  if (bad) { rumpy_set_error("rumpy_distill_bwd: %s", bad); return RUMPY_E_ARG; }
  if (p->rows == 0) return RUMPY_OK;
  const DsPlan plan = ds_plan(p->rows, p->V);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(p->rows * plan.splits));
  if (p->fmt == RUMPY_FMT_F32) hipLaunchKernelGGL((distill_bwd_kernel<RUMPY_FMT_F32>), grid, dim3(DS_WG), 0, s, *p, plan);
  else if (p->fmt == RUMPY_FMT_BF16) hipLaunchKernelGGL((distill_bwd_kernel<RUMPY_FMT_BF16>), grid, dim3(DS_WG), 0, s, *p, plan);
  else hipLaunchKernelGGL((distill_bwd_kernel<RUMPY_FMT_F16>), grid, dim3(DS_WG), 0, s, *p, plan);
  return rumpy_check_launch("rumpy_distill_bwd");
}
