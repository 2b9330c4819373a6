// Distillation from a teacher's top logits: the selection of the teacher's k largest logits of every row, the loss of a student against them,
// and the loss's gradient.  With u = z / tau, q = softmax(u) over all V columns, p the teacher's distribution over the columns it lists (and,
// when `tail` is given, the rest of the columns as one more outcome of probability p_t):
//   l = tau^2 [ sum_i p_i (log p_i - log q_i) + p_t (log p_t - log q_t) ],   q_t = sum of q over the columns that are not listed
//   dl/dz_j = tau (q_j - p_j) listed ;  tau q_j (1 - p_t / q_t) not listed       (no tail: p_t = 0, sum p = 1)
// Rows are [V] fp32 / bf16 / fp16 of a few classes, 8192 keys (the contrastive queue) or a few 100 000 columns.  Selection and loss read each row once (the
// selection's second look comes from registers), the gradient reads it once and writes it once: bound by memory, with one exponential per element
// and direction beside it.  The sum of exp runs over the row once with a running maximum per thread; q_t is summed directly over the columns
// that are not listed (a bit map of them lies in LDS): 1 - sum q_i would cancel where the listed columns hold nearly everything.
// The columns' exponentials and their sum are fp32; what is listed, a row's logarithms and joins and the sums over rows are 64-bit.  Every reduction has a
// fixed order, which goes with the call's sizes and the alignment of a row's address alone: results are bitwise reproducible.
#include "row_vec.hpp"

constexpr int DS_MAXK = 256, DS_MAXV = 1 << 30;
constexpr double LOG2E = 1.4426950408889634;
constexpr float LOG2E_F = (float)LOG2E;

__device__ __forceinline__ float wave_max(float v, int lane) {
  v = fmaxf(v, dpp_quad1(v)); v = fmaxf(v, dpp_quad2(v)); v = fmaxf(v, dpp_half_mirror(v)); v = fmaxf(v, dpp_row_mirror(v));
  v = fmaxf(v, lane_xor16(v, lane >> 4));
  return fmaxf(v, lane_xor32(v, lane));
}
// maximum over, and any of, the L neighbouring lanes of a row (16 or 64), in every one of them
template <int L> __device__ __forceinline__ float lanes_max(float v, int lane) {
  if constexpr (L == 64) return wave_max(v, lane);
  v = fmaxf(v, dpp_quad1(v)); v = fmaxf(v, dpp_quad2(v)); v = fmaxf(v, dpp_half_mirror(v));
  return fmaxf(v, dpp_row_mirror(v));
}
template <int L> __device__ __forceinline__ bool lanes_any(bool b, int lane) {
  const uint64_t all = __ballot(b);
  return (L == 64 ? all : all >> (lane & ~(L - 1)) & ((1ull << (L & 63)) - 1ull)) != 0ull;
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

// A launch has fewer than 2^32 threads along a dimension: calls of more rows than that holds (8.4 million at 512 threads a row) go in parts, each with the
// arguments of its own rows.  fn(first row, rows)
template <typename Fn> static void rows_in_parts(int64_t rows, int64_t threads_a_row, Fn fn) {
  const int64_t most = 0xffffff00ll / threads_a_row / 16 * 16;         // (whole workgroups of rows that share one)
  for (int64_t r = 0; r < rows; r += most) fn(r, rows - r < most ? rows - r : most);
}
static size_t elem_bytes(int fmt) { return fmt == RUMPY_FMT_F32 ? 4 : 2; }
template <typename T> static void advance(T*& p, int64_t bytes) { if (p) p = (T*)((const char*)p + bytes); }

// ================================================================================================================ selection
// order of the values as unsigned integers: -inf lowest, NaN highest, -0 = +0
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// (value, column) as one number: larger value first, then the lower column.  Never 0.
__device__ __forceinline__ uint64_t pair_of(float v, int col) { return ((uint64_t)order_key(v) << 32) | (uint32_t)~(uint32_t)col; }
__device__ __forceinline__ float pair_value(uint64_t p) { return key_value((uint32_t)(p >> 32)); }

constexpr int TL_WAVE_CAP = 256;      // candidates of a wave
constexpr float NOT_A_NUMBER = __builtin_nanf("");

// Rows that are few and long are cut: every piece of a row gives its own k largest pairs and its tail to a workspace, and one more workgroup per
// row joins them.
struct TlPlan { int splits, seg; float c; double inv_tau; };          // c = log2(e) / tau, rounded once
constexpr int TL_MOST_SPLITS = 32;
static TlPlan tl_plan(int64_t rows, int32_t V, double tau) {
  TlPlan p;
  p.c = (float)(LOG2E / tau);
  p.inv_tau = 1.0 / tau;
  int64_t s = 1;
  if (V >= 32768 && rows > 0) {
    s = (256 + rows - 1) / rows;
    const int64_t most = V / 8192;
    if (s > most) s = most;
    if (s > TL_MOST_SPLITS) s = TL_MOST_SPLITS;
  }
  p.seg = (int)((((int64_t)V + s - 1) / s + 63) / 64 * 64);
  p.splits = (int)(((int64_t)V + p.seg - 1) / p.seg);
  return p;
}

template <int WG> struct TlShared {
  static constexpr int WAVES = WG / 64;
  float red[WAVES];
  uint64_t cand[WAVES][TL_WAVE_CAP + 16];
  uint32_t count[WAVES];
  float after[WAVES * TL_WAVE_CAP];              // the candidates that are not chosen, by place
  uint32_t hist[256];
  uint32_t need;
  uint64_t prefix, kth, next;
};

// the value that `want` lanes of every wave reach with their `mine` (a bitwise search on ballots), the smallest of them over the waves: a bound that
// at least waves * want of the workgroup's values reach.  LOW: bits that only repeat the sign in this format's keys
template <int WG, int LOW> __device__ __forceinline__ uint32_t bound_of(uint32_t mine, int want, TlShared<WG>& sh) {
  uint32_t t = 0;
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t trial = t | (1u << bit);
    if (__popcll(__ballot(mine >= trial)) >= want) t = trial;
  }
  if (!(t & 0x80000000u)) t |= (1u << LOW) - 1u;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = __uint_as_float(t);
  __syncthreads();
  uint32_t b = __float_as_uint(sh.red[0]);
#pragma unroll
  for (int i = 1; i < WG / 64; ++i) b = min(b, __float_as_uint(sh.red[i]));
  return b;
}
// the value that k of the workgroup's `mine` reach: the same search over all waves, a barrier per bit (two buffers in turn, and one barrier in front: with fp16's
// LOW a search ends in the buffer that the next one begins with, and a row without a finite bound is searched twice)
template <int WG, int LOW> __device__ __forceinline__ uint32_t bound_of_all(uint32_t mine, int k, TlShared<WG>& sh) {
  uint32_t t = 0;
  __syncthreads();
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t trial = t | (1u << bit);
    uint32_t* n = sh.hist + (bit & 1) * (WG / 64);
    const uint64_t reach = __ballot(mine >= trial);
    if ((threadIdx.x & 63) == 0) n[threadIdx.x >> 6] = (uint32_t)__popcll(reach);
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < WG / 64; ++i) all += n[i];
    if (all >= (uint32_t)k) t = trial;
  }
  if (!(t & 0x80000000u)) t |= (1u << LOW) - 1u;
  return t;
}
// the k-th largest of `count` different pairs, 8 bits at a time from the top: needs no assumption about them
template <int WG, typename At> __device__ __forceinline__ uint64_t radix_kth(At at, int64_t count, int k, TlShared<WG>& sh) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) { sh.prefix = 0; sh.need = (uint32_t)k; }
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += WG) sh.hist[i] = 0;
    __syncthreads();
    const uint64_t prefix = sh.prefix, mask = shift == 56 ? 0ull : ~0ull << (shift + 8);
    const int64_t rounds = (count + WG - 1) / WG;
    for (int64_t i = 0; i < rounds; ++i) {                   // (whole waves: the ballots need every lane)
      const int64_t j = i * WG + tid;
      const uint64_t kk = j < count ? at(j) : 0;
      const bool in = j < count && (kk & mask) == prefix;
      const uint32_t bin = (uint32_t)(kk >> shift) & 255u;
      uint64_t left = __ballot(in);
      while (left) {                                       // one LDS add per distinct digit of the wave
        const int first = __ffsll((unsigned long long)left) - 1;
        const uint32_t b = __shfl(bin, first);
        const uint64_t same = __ballot(in && bin == b) & left;
        if ((tid & 63) == first) atomicAdd(&sh.hist[b], (uint32_t)__popcll(same));
        left &= ~same;
      }
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t need = sh.need, b = 255;
      while (b > 0 && sh.hist[b] < need) { need -= sh.hist[b]; --b; }
      sh.need = need;
      sh.prefix = prefix | ((uint64_t)b << shift);
    }
    __syncthreads();
  }
  return sh.prefix;
}
// Every wave keeps a list of its own in LDS, in the order of its walk: a place is the wave's count so far plus the hits in front in the wave, no atomics
// and nothing to wait for.  Called by whole waves.
template <int WG> __device__ __forceinline__ void push(bool hit, uint64_t p, uint32_t& count, TlShared<WG>& sh) {
  const uint64_t hits = __ballot(hit);
  if (hits) {
    const uint32_t at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0));
    if (hit && at < TL_WAVE_CAP) sh.cand[threadIdx.x >> 6][at] = p;
    count += (uint32_t)__popcll(hits);
  }
}
// closes the lists and puts each in order (by counting the larger pairs of the list, 16 at a time from LDS); returns the number of candidates, or
// ~0 where a list is too long
template <int WG> __device__ __forceinline__ uint32_t lists_done(uint32_t count, TlShared<WG>& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t* list = sh.cand[wave];
  if (count <= TL_WAVE_CAP) {
    if (lane < 16) list[count + lane] = 0;             // (no pair is 0)
    uint64_t mine[TL_WAVE_CAP / 64];
    uint32_t rank[TL_WAVE_CAP / 64];
#pragma unroll
    for (int i = 0; i < TL_WAVE_CAP / 64; ++i) {
      if (i * 64 >= count) break;
      mine[i] = i * 64 + lane < count ? list[i * 64 + lane] : 0;
      rank[i] = 0;
      for (uint32_t o = 0; o < count; o += 16) {
        uint64_t other[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) other[u] = list[o + u];
#pragma unroll
        for (int u = 0; u < 16; ++u) rank[i] += other[u] > mine[i];
      }
    }
#pragma unroll
    for (int i = 0; i < TL_WAVE_CAP / 64; ++i) {       // (a wave's LDS accesses stay in order: every pair is in a register by now)
      if (i * 64 >= count) break;
      if (i * 64 + lane < count) list[rank[i]] = mine[i];
    }
  }
  if (lane == 0) sh.count[wave] = count;
  __syncthreads();
  uint32_t n = 0;
  bool over = false;
#pragma unroll
  for (int w = 0; w < WG / 64; ++w) { n += sh.count[w]; over |= sh.count[w] > TL_WAVE_CAP; }
  return over ? ~0u : n;
}
// the candidates by their place among all: the place in the wave's own list and the larger pairs of the others, searched in all of them at once:
// emit(place, pair) for the first k; kth and next (0: there is none) for what comes after
template <int WG, typename Emit> __device__ __forceinline__ void place(int k, TlShared<WG>& sh, Emit emit) {
  constexpr int WAVES = WG / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) sh.next = 0;
  uint32_t most = 1;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) most = max(most, sh.count[w]);
  const uint32_t top = 1u << (31 - __clz((int)most));
  __syncthreads();
  for (uint32_t i = lane; i < sh.count[wave]; i += 64) {
    const uint64_t mine = sh.cand[wave][i];
    uint32_t in_front[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) in_front[w] = 0;
    for (uint32_t b = top; b; b >>= 1) {
      uint64_t other[WAVES];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) other[w] = sh.cand[w][min(in_front[w] + b, (uint32_t)TL_WAVE_CAP) - 1];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) if (in_front[w] + b <= sh.count[w] && other[w] > mine) in_front[w] += b;
    }
    uint32_t rank = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) rank += in_front[w];
    if (rank < (uint32_t)k) {
      emit((int)rank, mine);
      if (rank == (uint32_t)k - 1) sh.kth = mine;
    } else {
      sh.after[rank] = pair_value(mine);
      if (rank == (uint32_t)k) sh.next = mine;
    }
  }
  __syncthreads();
}

// A row (or a piece of one) as whole 16-byte pieces of 8 elements at aligned addresses, and up to 7 elements in front and behind (a row of odd
// length starts anywhere: pieces at odd addresses run at two thirds of the rate).  NP > 1: a thread's first NP pieces stay in registers, so that
// they are read once; what a longer row has beyond comes from the caches at every look.  NP 1: rows of at most 8 WG elements, element by element over the threads (pieces would leave waves without any).
template <int FMT, int WG, int NP> struct RowPieces {
  typedef typename RowElem<FMT>::type E;
  const E* z;
  int len, head, count, tailn;
  RowRaw<FMT> raw[NP > 1 ? NP : 1];
  E one[NP == 1 ? 8 : 1];
  __device__ __forceinline__ RowPieces(const E* z_, int len_) : z(z_), len(len_) {
    head = min(len, (int)((16u - (uint32_t)(uintptr_t)z % 16u) % 16u / (uint32_t)sizeof(E)));
    count = (len - head) / 8;
    tailn = len - head - 8 * count;
  }
  __device__ __forceinline__ void load() {
    if constexpr (NP > 1) {
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        if (u * WG >= count) break;
        raw[u] = load_piece<FMT>(z + head + 8 * min(u * WG + (int)threadIdx.x, count - 1), 8, 0.f);
      }
    } else if constexpr (NP == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = z[min(i * WG + (int)threadIdx.x, len - 1)];
    }
  }
  // fn(8 values, column of the first, columns from one to the next), by whole waves; what lies outside the row is -inf
  template <typename Fn> __device__ __forceinline__ void each(Fn fn) const {
    float v[8];
    if constexpr (NP == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i * WG + (int)threadIdx.x < len ? elem_to_f32<FMT>(one[i]) : -INFINITY;
      fn(v, (int)threadIdx.x, WG);
      return;
    }
    if constexpr (NP > 1) {
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        if (u * WG >= count) break;
        unpack_piece<FMT>(raw[u], v);
        const int p = u * WG + (int)threadIdx.x;
        if ((u + 1) * WG > count) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = p < count ? v[i] : -INFINITY;
        }
        fn(v, head + 8 * p, 1);
      }
    }
    if (NP * WG < count) {
      auto piece = [&](int p) { return load_piece<FMT>(z + head + (size_t)8 * min(p, count - 1), 8, 0.f); };
      RowRaw<FMT> next = piece(NP * WG + (int)threadIdx.x);
      for (int p0 = NP * WG; p0 < count; p0 += WG) {
        const int p = p0 + (int)threadIdx.x;
        unpack_piece<FMT>(next, v);
        next = piece(p + WG);
        if (p0 + WG > count) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = p < count ? v[i] : -INFINITY;
        }
        fn(v, head + 8 * p, 1);
      }
    }
    if (threadIdx.x < 64 && head + tailn) {          // the ends: lanes 0 and 1
      const int first = threadIdx.x == 0 ? 0 : len - tailn, n = threadIdx.x == 0 ? head : threadIdx.x == 1 ? tailn : 0;
      unpack_piece<FMT>(load_piece<FMT>(z + first, n, -INFINITY), v);
      fn(v, first, 1);
    }
  }
};

// log sum exp(z / tau) over the elements whose pair lies under `kth`, by their maximum; every thread gets it
template <int FMT, int WG> __device__ __forceinline__ float rest_below(const RowPieces<FMT, WG, 0>& row, uint64_t kth, const TlPlan& plan, float* red) {
  const float c = plan.c;
  float rmx = -INFINITY, bad = 0.f;
  row.each([&](const float (&v)[8], int j, int stride) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (pair_of(v[i], j + i * stride) < kth) { rmx = fmaxf(rmx, v[i]); if (v[i] != v[i]) bad = 1.f; }
  });
  rmx = block_max<WG / 64>(rmx, red);
  if (block_max<WG / 64>(bad, red) > 0.f) return NOT_A_NUMBER;
  if (!(fabsf(rmx) < INFINITY)) return rmx;
  float s = 0.f;
  row.each([&](const float (&v)[8], int j, int stride) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s += __builtin_amdgcn_exp2f(pair_of(v[i], j + i * stride) < kth ? (v[i] - rmx) * c : -INFINITY);
  });
  return (float)(rmx * plan.inv_tau + log(block_sum<WG / 64>(s, red)));
}

// One workgroup per row or piece, two looks at it: a bound T that at least k elements reach, from every thread's maximum; then the few elements
// that reach the bound (a few times k) and the sum of exp over all others.  Where that does not do - too many reach the bound (columns of equal
// value), it is infinite or a type's lowest value (fewer than about k columns that no mask holds), or there is NaN - the elements above T and, as
// far as they do not suffice, those equal to it in the lowest columns; and where those are too many as well, the k-th pair by radix search.
// Measured (MI355X): 2048 x 65521 bf16, k 100: 73 us = 3.7 TB/s (k 1: 62); 4096 x 8192 bf16, k 64: 28 us; 16384 x 1000 fp32, k 64: 37 us, k 4: 15; 32 x 8192
// fp32: 8 us, one row's chain of latencies.  256 x 65521: 18 us; with 100 valid columns, constant, or with its largest in the first 1000: 34 - 50 us (by radix search: 430 - 560; ascending
// rows still go that way).
// Six waves a SIMD: three workgroups of 512 a CU, with most of a row each in registers (with two, 2048 rows of 65521 took 80 us instead of 70).
template <int FMT, int WG, int NP> __global__ void __launch_bounds__(WG, 6) top_logits_kernel(rumpy_top_logits_args a, TlPlan plan) {
  typedef typename RowElem<FMT>::type E;
  __shared__ TlShared<WG> sh;
  const int tid = threadIdx.x;
  const float c = plan.c;
  const int64_t row = blockIdx.x / plan.splits;
  const int piece = blockIdx.x % plan.splits, c0 = piece * plan.seg;
  RowPieces<FMT, WG, NP> r(reinterpret_cast<const E*>(a.logits) + (size_t)row * a.ld + c0, min(plan.seg, a.V - c0));
  r.load();
  // the rare ways read the row again, in loops: unrolled over registers like the two looks they made the kernel 10 us slower for every row
  const RowPieces<FMT, WG, 0> again(r.z, r.len);
  const int len = r.len, k = min(a.k, len);
  uint32_t n = ~0u, mine = 0;                             // candidates of the row (~0: a list is too long), of the wave
  float T = 0.f, sum = 0.f;
  bool summed = false;                                    // `sum` holds everything under T
  if (NP == 1 && len <= WG) {                             // one element per thread: all of them are candidates
    push(tid < len, pair_of(elem_to_f32<FMT>(r.one[0]), tid), mine, sh);
    n = lists_done(mine, sh);
    summed = true;
  } else {
    constexpr int LOW = FMT == RUMPY_FMT_BF16 ? 16 : FMT == RUMPY_FMT_F16 ? 13 : 0;
    auto usable = [&](float b) { return fabsf(b * c) < INFINITY && fabsf(b) < INFINITY; };
    float mx = -INFINITY;                                 // (NaN is passed over here; the second look meets it)
    r.each([&](const float (&v)[8], int, int) {
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, v[i]);
    });
    T = key_value(bound_of<WG, LOW>(order_key(mx), (k + WG / 64 - 1) / (WG / 64), sh));
    // (masked columns may leave a wave without enough of its own)
    if (!usable(T)) T = key_value(bound_of_all<WG, LOW>(order_key(mx), k, sh));
    if (usable(T)) {
      const float m = T * c;
      r.each([&](const float (&v)[8], int j, int stride) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool hit = v[i] >= T;
          any |= hit;
          sum += __builtin_amdgcn_exp2f(fmaf(hit ? -INFINITY : v[i], c, -m));
        }
        if (__ballot(any)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) push(v[i] >= T, pair_of(v[i], j + i * stride), mine, sh);
        }
      });
      sum = block_sum<WG / 64>(sum, sh.red);
      n = lists_done(mine, sh);
      summed = n != ~0u && sum == sum;
    }
    if (!summed) {
      T = key_value(bound_of_all<WG, LOW>(order_key(mx), k, sh));
      mine = 0;
      again.each([&](const float (&v)[8], int j, int stride) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) any |= !(v[i] <= T);            // (NaN counts as largest)
        if (__ballot(any)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) push(!(v[i] <= T), pair_of(v[i], j + i * stride), mine, sh);
        }
      });
      n = lists_done(mine, sh);
      if (n < (uint32_t)k) {
        // in the order of the columns, WG of them a round, until there are enough
        int turn = 0;
        for (int j0 = 0; j0 < len && n < (uint32_t)k; j0 += WG, turn ^= 1) {
          const int j = j0 + tid;
          const float v = elem_to_f32<FMT>(r.z[min(j, len - 1)]);
          push(j < len && v == T, pair_of(v, j), mine, sh);
          uint32_t* counts = sh.hist + turn * (WG / 64);
          if ((tid & 63) == 0) counts[tid >> 6] = mine;
          __syncthreads();
          n = 0;
#pragma unroll
          for (int w = 0; w < WG / 64; ++w) n += counts[w];
        }
        n = lists_done(mine, sh);
      }
    }
  }
  if (n == ~0u) {
    const uint64_t kth = radix_kth([&](int64_t j) { return pair_of(elem_to_f32<FMT>(r.z[j]), (int)j); }, len, k, sh);      // exactly k pairs reach it
    mine = 0;
    for (int j0 = 0; j0 < len; j0 += WG) {
      const int j = j0 + tid;
      const uint64_t p = pair_of(elem_to_f32<FMT>(r.z[min(j, len - 1)]), j);
      push(j < len && p >= kth, p, mine, sh);
    }
    n = lists_done(mine, sh);
  }
  uint64_t* pairs = plan.splits > 1 ? (uint64_t*)a.work + (size_t)blockIdx.x * a.k : nullptr;
  place(k, sh, [&](int at, uint64_t p) {
    const uint32_t col = ~(uint32_t)p;
    if (pairs) pairs[at] = p - (uint32_t)c0;               // ~(col + c0) = ~col - c0
    else {
      reinterpret_cast<E*>(a.values)[(size_t)row * a.k + at] = r.z[col];
      reinterpret_cast<int64_t*>(a.indices)[(size_t)row * a.k + at] = col;
    }
  });
  if (pairs) for (int i = k + tid; i < a.k; i += WG) pairs[i] = 0;       // a piece shorter than k
  float tail;
  if (n == (uint32_t)len && sh.next == 0) tail = -INFINITY;      // everything is chosen
  else if (!summed || (sh.next == 0 && sum < 1e-20f)) {
    // no sum was made, or nothing was collected beyond the top and the others lie so far under the bound that their sum has no digits left
    tail = rest_below(again, sh.kth, plan, sh.red);
  } else {
    const float next = sh.next ? pair_value(sh.next) : T;
    // relative to the largest that was not chosen: the other candidates, and the sum under the bound with T's distance from it
    float s = 0.f;
    for (uint32_t i = k + tid; i < n; i += WG) s += __builtin_amdgcn_exp2f((sh.after[i] - next) * c);
    s = block_sum<WG / 64>(s, sh.red) + (sum > 0.f ? sum * __builtin_amdgcn_exp2f((T - next) * c) : 0.f);
    tail = fabsf(next) < INFINITY ? (float)(next * plan.inv_tau + logf(s)) : next;
  }
  if (tid == 0) {
    if (pairs) reinterpret_cast<float*>((uint64_t*)a.work + (size_t)gridDim.x * a.k)[blockIdx.x] = tail;
    else a.tail[row] = tail;
  }
}

// the pieces' pairs (each list in order) to the row's k, by the same two steps; what is left of them joins the pieces' tails.  All pairs are in
// registers; consecutive threads take the same place of consecutive lists, so that what is collected spreads over the waves.
template <int FMT> __global__ void __launch_bounds__(512) top_join_kernel(rumpy_top_logits_args a, TlPlan plan) {
  typedef typename RowElem<FMT>::type E;
  constexpr int WG = 512, NP = TL_MOST_SPLITS * DS_MAXK / WG;
  __shared__ TlShared<WG> sh;
  const int tid = threadIdx.x, k = a.k, S = plan.splits, count = S * k;
  const int64_t row = blockIdx.x;
  const E* z = reinterpret_cast<const E*>(a.logits) + (size_t)row * a.ld;
  const uint64_t* pairs = (const uint64_t*)a.work + (size_t)row * count;
  const float* tails = reinterpret_cast<const float*>((const uint64_t*)a.work + (size_t)gridDim.x * count) + (size_t)row * S;
  uint64_t mine[NP];
#pragma unroll
  for (int u = 0; u < NP; ++u) {
    const int j = u * WG + tid;
    mine[u] = j < count ? pairs[(j % S) * k + j / S] : 0;
  }
  const float tail_in = tid < S ? tails[tid] : -INFINITY;
  // the bound: of every list the pair that ceil(k / lists) of its pairs reach, the smallest of them
  if (tid == 0) sh.prefix = ~0ull;
  __syncthreads();
  if (tid < S) atomicMin((unsigned long long*)&sh.prefix, (unsigned long long)pairs[tid * k + (k + S - 1) / S - 1]);
  __syncthreads();
  const uint64_t bound = sh.prefix;
  auto gather = [&](uint64_t from) {
    uint32_t listed = 0;
#pragma unroll
    for (int u = 0; u < NP; ++u) push(mine[u] && mine[u] >= from, mine[u], listed, sh);
    return lists_done(listed, sh);
  };
  uint32_t n = gather(bound);
  if (n == ~0u || n < (uint32_t)k) {                   // (fewer than k: the last list is short)
    const uint64_t kth = radix_kth([&](int64_t j) { return pairs[j]; }, count, k, sh);
    n = gather(kth);
  }
  place(k, sh, [&](int at, uint64_t p) {
    const uint32_t col = ~(uint32_t)p;
    reinterpret_cast<E*>(a.values)[(size_t)row * k + at] = z[col];
    reinterpret_cast<int64_t*>(a.indices)[(size_t)row * k + at] = col;
  });
  const uint64_t kth = sh.kth;
  float m = tail_in, bad = tail_in != tail_in ? 1.f : 0.f;
#pragma unroll
  for (int u = 0; u < NP; ++u) {
    if (mine[u] && mine[u] < kth) {
      const float v = (float)(pair_value(mine[u]) * plan.inv_tau);
      m = fmaxf(m, v);
      if (v != v) bad = 1.f;
    }
  }
  m = block_max<WG / 64>(m, sh.red);
  bad = block_max<WG / 64>(bad, sh.red);
  float s = __builtin_amdgcn_exp2f((tail_in - m) * LOG2E_F);
#pragma unroll
  for (int u = 0; u < NP; ++u) {
    if (mine[u] && mine[u] < kth) s += __builtin_amdgcn_exp2f(((float)(pair_value(mine[u]) * plan.inv_tau) - m) * LOG2E_F);
  }
  s = block_sum<WG / 64>(s, sh.red);
  if (tid == 0) a.tail[row] = bad > 0.f ? NOT_A_NUMBER : fabsf(m) < INFINITY ? m + logf(s) : m;
}

extern "C" int64_t rumpy_top_logits_work_bytes(int64_t rows, int32_t V, int32_t k) {
  if (rows <= 0 || V < 1 || V > DS_MAXV || k < 1 || k > DS_MAXK) return 0;
  const TlPlan plan = tl_plan(rows, V, 1.0);
  return plan.splits > 1 ? rows * plan.splits * (k * 8 + 4) : 0;
}
template <int FMT, int WG> static void tl_launch_wg(const rumpy_top_logits_args& a, const TlPlan& plan, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * plan.splits)), wg(WG);
  const int len = a.V < plan.seg ? a.V : plan.seg, np = (len / 8 + WG - 1) / WG;
  // pieces in registers: the callers' limits, and 60 registers at 512 threads.  (fp32 at 256 threads: 8 pieces are 64 registers of the 80 that six waves leave, 36 others
  // lie in scratch: 4096 x 16384, k 64, 56 us = 4.8 TB/s.)
  constexpr int MOST = WG <= 128 ? 4 : WG == 256 ? 8 : FMT == RUMPY_FMT_F32 ? 7 : 15;
  if (len <= 8 * WG) hipLaunchKernelGGL((top_logits_kernel<FMT, WG, 1>), grid, wg, 0, s, a, plan);
  else if (np <= 2) hipLaunchKernelGGL((top_logits_kernel<FMT, WG, 2>), grid, wg, 0, s, a, plan);
  else if (np <= 4) hipLaunchKernelGGL((top_logits_kernel<FMT, WG, 4>), grid, wg, 0, s, a, plan);
  else if (np <= 8 && MOST > 8) hipLaunchKernelGGL((top_logits_kernel<FMT, WG, (MOST > 8 ? 8 : MOST)>), grid, wg, 0, s, a, plan);
  else hipLaunchKernelGGL((top_logits_kernel<FMT, WG, MOST>), grid, wg, 0, s, a, plan);
}
// (rows that are cut are few: never in parts)
template <int FMT, int WG> static void tl_launch_parts(const rumpy_top_logits_args& a, const TlPlan& plan, hipStream_t s) {
  rows_in_parts(a.rows, (int64_t)WG * plan.splits, [&](int64_t r, int64_t n) {
    rumpy_top_logits_args b = a;
    const int64_t e = elem_bytes(FMT);
    b.rows = n;
    advance(b.logits, r * a.ld * e); advance(b.values, r * a.k * e); advance(b.indices, r * a.k * 8); advance(b.tail, r * 4);
    tl_launch_wg<FMT, WG>(b, plan, s);
  });
}
template <int FMT> static void tl_launch(const rumpy_top_logits_args& a, const TlPlan& plan, hipStream_t s) {
  // Short rows: small workgroups, more rows at once (a row is a chain of latencies: bound, lists, places) and no barriers in one of 64.  At least 2 k threads,
  // so that the bound comes from the better half of the threads' maxima (with k threads the lists run over: 65536 x 1000, k 64: 808 us with 64).
  // us, bf16, 64 | 128 | 256 | 512 threads a row:  65536 x 300, k 16: 47 | 85 | 178 | 414     16384 x 1000, k 4: 15 | 23 | 46 | 112
  // 4096 x 1000, k 64: - | 14 | 18 | 37     4096 x 4000, k 48: - | 17 | 22 | 38     4096 x 8000, k 96: - | - | 33 | 48     4096 x 600, k 192: - | - | 39 | 49
  // 32 x 1000, k 4: 4.8 | 4.7 | 5.2 | 6.8     32 x 4000, k 64: - | 9.7 | 6.5 | 6.6     32 x 16000, k 64: - | - | 10 | 8
  const bool few = a.rows < 256, many = a.rows >= 1024;
  if (a.k <= 32 && a.V <= (many ? 2048 : 1024)) tl_launch_parts<FMT, 64>(a, plan, s);
  else if (a.k <= 64 && a.V <= (many ? 4096 : 2048)) tl_launch_parts<FMT, 128>(a, plan, s);
  else if (few ? a.k <= 96 && a.V <= 4096 : a.k <= 128 ? a.V <= 16384 : many && a.k <= 192 && a.V <= 2048) tl_launch_parts<FMT, 256>(a, plan, s);
  else tl_launch_parts<FMT, 512>(a, plan, s);
  if (plan.splits > 1) hipLaunchKernelGGL((top_join_kernel<FMT>), dim3((unsigned)a.rows), dim3(512), 0, s, a, plan);
}
extern "C" int rumpy_top_logits(const rumpy_top_logits_args* p, void* stream) {
  const char* bad = !p ? "no arguments" : nullptr;
  if (!bad && (p->fmt != RUMPY_FMT_F32 && p->fmt != RUMPY_FMT_BF16 && p->fmt != RUMPY_FMT_F16)) bad = "fp32, bf16 or fp16 logits";
  if (!bad && (p->rows < 0 || p->V < 1 || p->V > DS_MAXV || p->ld < 0)) bad = "rows of 1 .. 2^30 logits";
  if (!bad && (p->k < 1 || p->k > DS_MAXK || p->k > p->V)) bad = "1 .. 256 top logits, no more than the row has";
  if (!bad && !(p->tau >= 1e-30 && p->tau <= 1e30)) bad = "a temperature above zero";
  if (!bad && p->rows && (!p->logits || !p->values || !p->indices || !p->tail)) bad = "a tensor is missing";
  if (!bad && rumpy_top_logits_work_bytes(p->rows, p->V, p->k) && (!p->work || ((uintptr_t)p->work & 7)))
    bad = "rows of this length and number are cut and need `work` (rumpy_top_logits_work_bytes, at a multiple of 8)";
  if (!bad && p->rows > 0x7fffffff) bad = "at most 2^31 - 1 rows";
  if (bad) { rumpy_set_error("rumpy_top_logits: %s", bad); return RUMPY_E_ARG; }
  if (p->rows == 0) return RUMPY_OK;
  const TlPlan plan = tl_plan(p->rows, p->V, p->tau);
  hipStream_t s = (hipStream_t)stream;
  if (p->fmt == RUMPY_FMT_F32) tl_launch<RUMPY_FMT_F32>(*p, plan, s);
  else if (p->fmt == RUMPY_FMT_BF16) tl_launch<RUMPY_FMT_BF16>(*p, plan, s);
  else tl_launch<RUMPY_FMT_F16>(*p, plan, s);
  return rumpy_check_launch("rumpy_top_logits");
}

// ================================================================================================================ loss and gradient
constexpr int DS_WG = 512, DS_WAVES = DS_WG / 64;
constexpr int DS_STATE = 8;      // per row: reference and coefficient of the streamed columns, maximum of all and 1 / sum, the teacher's factor beside its maximum, dead, the
                                 // teacher's maximum, whether a column may be listed twice
constexpr double DS_LEAST = -126.0 / LOG2E;      // exponents below it count as 0, as the columns' own do

// exp((v - m) / tau), v <= m, with c + lo = log2(e) / tau: c alone, rounded to 32 bits, is another temperature for the whole row, and its error of up to
// 2^-25 does not average out in the loss (1.8e-6 of it where 32-bit divisions made 2e-7).  The difference first: no digits are lost where a row lies
// far from zero, and none of it overflows (lowest values of a type as masks).  v = -inf gives 0, which is why lo is positive; m is finite.
__device__ __forceinline__ float ds_exp(float v, float m, float c, float lo) {
  const float d = v - m;
  return __builtin_amdgcn_exp2f(fmaf(d, lo, d * c));
}
// the factor from a sum relative to m to one relative to M >= m (m = -inf: there is no sum yet; M = inf: NaN, by the sum itself)
__device__ __forceinline__ float ds_rescale(float m, float M, float c, float lo) { return m == -INFINITY ? 0.f : m == M ? 1.f : ds_exp(m, M, c, lo); }

struct DsPlan { int splits, seg; float c, lo, near; double inv_tau; };      // c + lo = log2(e) / tau; near: the nearest float to it
// rows are cut when there are too few of them to fill the chip; a piece's bit map of listed columns has to fit LDS (2^18 columns: 32 KB)
static DsPlan ds_plan(int64_t rows, int32_t V, double tau) {
  DsPlan p;
  // c is rounded towards zero: a -inf (a masked column) times c and times a positive lo is -inf, where a negative lo would make it NaN
  const double x = LOG2E / tau;
  p.near = (float)x;
  p.c = (double)p.near > x ? nextafterf(p.near, 0.f) : p.near;
  p.lo = fmaxf((float)(x - p.c), p.c * 1e-12f);
  p.inv_tau = 1.0 / tau;
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
struct DsListed { int idx[DS_MAXK]; float v[DS_MAXK]; float z[DS_MAXK]; bool first[DS_MAXK]; };
template <int FMT> __device__ __forceinline__ int ds_load_listed(const rumpy_distill_args& a, int64_t row, const typename RowElem<FMT>::type* z, DsListed& l) {
  const int tid = threadIdx.x;
  int mine = -1;
  if (tid < a.k) {
    const int64_t i = ds_index(a, row, tid);
    const bool inside = i >= 0 && i < a.V;
    mine = i < 0 ? -1 : inside ? (int)i : -2;
    l.idx[tid] = mine;
    l.v[tid] = ds_value(a, row, tid);
    l.z[tid] = inside ? elem_to_f32<FMT>(z[i]) : 0.f;
  }
  __syncthreads();
  // (16 at a time, from LDS whole: one by one every look waits for the one before it - 20 us for 256 entries)
  if (a.tail && tid < a.k) {
    bool f = true;
    for (int o = 0; o < a.k; o += 16) {
      int other[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) other[i] = l.idx[o + i];
#pragma unroll
      for (int i = 0; i < 16; ++i) f &= !(o + i < tid && other[i] == mine);
    }
    l.first[tid] = f;
  }
  return mine;
}

// sum over the L neighbouring lanes of a row (16 or 64), in every one of them: lanes_sum's order in 64 bits
template <typename Move> __device__ __forceinline__ double moved(double v, Move move) {
  return __hiloint2double(__float_as_int(move(__int_as_float(__double2hiint(v)))), __float_as_int(move(__int_as_float(__double2loint(v)))));
}
template <int L> __device__ __forceinline__ double lanes_sum64(double v, int lane) {
  v += moved(v, dpp_quad1); v += moved(v, dpp_quad2); v += moved(v, dpp_half_mirror); v += moved(v, dpp_row_mirror);
  if constexpr (L == 64) {
    v += moved(v, [&](float x) { return lane_xor16(x, lane >> 4); });
    v += moved(v, [&](float x) { return lane_xor32(x, lane); });
  }
  return v;
}

// L lanes of one wave: the row's loss and what its gradient needs, from the sum over the streamed columns (all of them, or the unlisted ones when the
// rest is an outcome): s = sum exp((z - m) / tau).  With the rest as an outcome the loss is of second order in the difference of the two distributions,
// and so is all that s's rounding costs it as long as each distribution sums to 1: what is listed and the joined sums are made in 64 bits.  (In 32 bits they
// left an error of the first order: 2^-24 tau^2, 5e-4 of the loss of 3 x 168911 columns, 1 listed, tau 4, where it is 2e-7 now; 65536 x 100, 8 listed: 20 us
// then, 23 now; 16384 x 1000 17 and 18.)
// idx, v, z: what the teacher lists, in LDS; first(i): no earlier entry names entry i's column; doubled: some column may be named twice.
template <int L, typename First>
__device__ __forceinline__ void ds_finish(const rumpy_distill_args& a, const DsPlan& plan, int64_t row, const int* idx, const float* v, const float* z, First first,
                                          bool doubled, float m, float s, int lane) {
  const double inv_tau = plan.inv_tau;
  const bool rest = a.tail != nullptr;
  const float w = a.row_weight ? a.row_weight[row] : 1.f;
  float vm = -INFINITY, zm = -INFINITY;
  bool odd = false, outside = false;
  for (int i = lane % L; i < a.k; i += L) {
    if (idx[i] == -1) continue;
    outside |= idx[i] == -2;
    odd |= v[i] != v[i];
    vm = fmaxf(vm, v[i]);
    zm = fmaxf(zm, z[i]);
  }
  vm = lanes_max<L>(vm, lane);
  zm = lanes_max<L>(zm, lane);
  const float tl = rest ? a.tail[row] : -INFINITY;
  bool nan = lanes_any<L>(odd || outside, lane) || tl != tl;
  float* st = a.state + row * DS_STATE;
  if (!nan && vm == -INFINITY && tl == -INFINITY) {            // the teacher says nothing about this row
    if (lane % L == 0) { a.row_loss[row] = 0.f; st[0] = st[1] = st[2] = st[3] = st[4] = 0.f; st[5] = 1.f; }
    return;
  }
  // the teacher's logarithms relative to its largest logit, so that far from zero no digits are lost: log p = (v - vm) / tau - up - log P
  // (up: the tail where it is the larger, or all there is)
  const bool tail_alone = vm == -INFINITY;
  if (tail_alone) vm = 0.f;
  const double tr = tl - vm * inv_tau, up = tr > 0.0 || tail_alone ? tr : 0.0;
  const float M = rest ? fmaxf(m, zm) : m;
  double p_listed = 0.0, q_listed = 0.0, loss = 0.0;          // sums of the listed p and q up to the factors 1 / P and 1 / S, and of p times the difference of their exponents
  for (int i = lane % L; i < a.k; i += L) {
    if (idx[i] < 0) continue;
    const double lp = ((double)v[i] - vm) * inv_tau - up, lq = ((double)z[i] - M) * inv_tau;
    if (!(lp < DS_LEAST)) {
      const double e = exp(lp);
      p_listed += e;
      loss += e * (lp - lq);
    }
    if (rest && first(i)) q_listed += exp(lq);
  }
  p_listed = lanes_sum64<L>(p_listed, lane);
  loss = lanes_sum64<L>(loss, lane);
  // (the row's three exponentials, and its three logarithms, in three lanes at once: one after another the logarithms were a third of a short row's time)
  const double to_m = m == -INFINITY ? (double)-INFINITY : ((double)m - M) * inv_tau, to_rest = tr - up;
  double P = p_listed, S = s, p_rest = 0.0, q_rest = 0.0, beside = 1.0;          // beside: of the listed entries' exponents, relative to the teacher's largest logit
  if (rest) {
    const double ex = exp(lane % 4 == 0 ? to_rest : lane % 4 == 1 ? to_m : -up);
    p_rest = to_rest < DS_LEAST ? 0.0 : __shfl(ex, 0, L);
    q_rest = m == -INFINITY ? 0.0 : s * __shfl(ex, 1, L);
    beside = __shfl(ex, 2, L);
    P += p_rest;
    S = lanes_sum64<L>(q_listed, lane) + q_rest;
  }
  // (infinite logits of the teacher; NaN in the streamed columns, which their maximum passes over: m may be -inf beside it)
  nan |= P != P || s != s;
  const double ln = log(lane % 4 == 0 ? P : lane % 4 == 1 ? S : (double)s);
  const double ln_p = __shfl(ln, 0, L), ln_s = __shfl(ln, 1, L), ln_r = __shfl(ln, 2, L), one_p = 1.0 / P, one_s = 1.0 / S;
  loss = (loss - p_listed * (ln_p - ln_s)) * one_p;
  float coef = (float)one_s;
  if (rest) {
    if (p_rest != 0.0) loss += p_rest * one_p * ((to_rest - ln_p) - (to_m + ln_r - ln_s));
    coef = m == -INFINITY ? 0.f : (float)(q_rest * one_s - p_rest * one_p) / s;
  }
  if (nan) loss = coef = NOT_A_NUMBER;
  if (lane % L == 0) {
    a.row_loss[row] = w == 0.f ? 0.f : (float)(w * loss * a.tau * a.tau);
    st[0] = m == -INFINITY ? 0.f : m;
    st[1] = coef;
    st[2] = M;
    st[3] = nan ? coef : (float)one_s;
    st[4] = tail_alone ? 0.f : (float)(beside * one_p);
    st[5] = w == 0.f ? 1.f : 0.f;
    st[6] = vm;
    st[7] = doubled ? 1.f : 0.f;
  }
}

// One workgroup per piece of a row.  REST: the listed columns are left out of the sum (bit map in LDS).
// Measured (MI355X): 4096 x 50021 bf16 95 us = 4.3 TB/s (80 without REST and the second part of the temperature; 139 with one piece in flight at odd
// addresses), 1000 x 32000 fp32 22 us, 32 x 8192 fp32 9 us.
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
  // whole pieces lie at 16-byte addresses (RowPieces); their bits at whole bytes: column j of the piece of the row has bit j - j0 + shift
  const RowPieces<FMT, DS_WG, 0> r(z + j0, (int)(j1 - j0));
  const int shift = (8 - r.head) & 7, body = r.head ? 1 : 0;
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bits);
  // U pieces are asked for before the U before them are summed (the first before anything else); their maximum is joined once
  constexpr int U = FMT == RUMPY_FMT_F32 ? 2 : 4;
  RowRaw<FMT> raw[U];
  const int whole = r.count / (DS_WG * U);             // rounds in which every thread has U whole pieces
  const E* zp = r.z + r.head + tid * 8;
  if (whole) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_piece<FMT>(zp + u * DS_WG * 8, 8, 0.f);
  }
  if constexpr (REST) {
    const int words = (r.len + 7 + 31) / 32;
    for (int i = tid; i < words; i += DS_WG) bits[i] = 0;
    if (plan.splits > 1) __syncthreads();
  }
  int64_t mine = -1;
  if (plan.splits == 1) mine = ds_load_listed<FMT>(a, row, z, l);      // (holds a barrier)
  else if (REST && tid < a.k) mine = ds_index(a, row, tid);
  if constexpr (REST) {
    if (mine >= j0 && mine < j1) { const int bit = (int)(mine - j0) + shift; atomicOr(&bits[bit >> 5], 1u << (bit & 31)); }
    __syncthreads();
  }
  const float c = plan.c, lo = plan.lo;
  float m = -INFINITY, ref = 0.f, s = 0.f;            // ref: m, or 0 as long as there is nothing but -inf
  auto sum_up = [&](auto& v) {
    constexpr int N = sizeof(v) / sizeof(v[0]);
    float top = v[0][0];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, v[u][i]);
    if (top > m) {
      s *= ds_rescale(m, top, c, lo);
      m = ref = top;
    }
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += ds_exp(v[u][i], ref, c, lo);
  };
  auto leave_out = [&](float (&v)[8], uint32_t here) {
    if (here) {
#pragma unroll
      for (int i = 0; i < 8; ++i) if (here >> i & 1u) v[i] = -INFINITY;
    }
  };
  for (int b = 0; b < whole; ++b) {
    float v[U][8];
    uint32_t here[U];
    if constexpr (REST) {
#pragma unroll
      for (int u = 0; u < U; ++u) here[u] = bytes[(b * U + u) * DS_WG + tid + body];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) unpack_piece<FMT>(raw[u], v[u]);
    const E* next = zp + (size_t)min(b + 1, whole - 1) * (DS_WG * 8 * U);
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_piece<FMT>(next + u * DS_WG * 8, 8, 0.f);
    if constexpr (REST) {
#pragma unroll
      for (int u = 0; u < U; ++u) leave_out(v[u], here[u]);
    }
    sum_up(v);
  }
  for (int p0 = whole * DS_WG * U; p0 < r.count; p0 += DS_WG) {
    const int p = p0 + tid;
    float v[1][8];
    unpack_piece<FMT>(load_piece<FMT>(r.z + r.head + (size_t)8 * min(p, r.count - 1), 8, 0.f), v[0]);
    leave_out(v[0], p >= r.count ? 0xffu : REST ? bytes[p + body] : 0u);
    sum_up(v);
  }
  if (tid < 64 && r.head + r.tailn) {                  // the ends: lanes 0 and 1
    const int first = tid == 0 ? 0 : r.len - r.tailn, n = tid == 0 ? r.head : tid == 1 ? r.tailn : 0;
    float v[1][8];
    unpack_piece<FMT>(load_piece<FMT>(r.z + first, n, -INFINITY), v[0]);
    if constexpr (REST) {
#pragma unroll
      for (int i = 0; i < 8; ++i) { const int bit = first + i + shift; if (i < n && (bytes[bit >> 3] >> (bit & 7) & 1u)) v[0][i] = -INFINITY; }
    }
    sum_up(v);
  }
  const float M = block_max<DS_WAVES>(m, red);
  s = block_sum<DS_WAVES>(m == -INFINITY ? s : s * ds_rescale(m, M, c, lo), red);
  if (plan.splits > 1) {
    if (tid == 0) { a.partial[blockIdx.x * (size_t)2] = M; a.partial[blockIdx.x * (size_t)2 + 1] = s; }
    return;
  }
  if (tid < 64) ds_finish<64>(a, plan, row, l.idx, l.v, l.z, [&](int i) { return l.first[i]; }, true, M, s, tid);
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
  const float c = plan.c, lo = plan.lo;
  const float* part = a.partial + (size_t)row * plan.splits * 2;
  float m = -INFINITY;
  for (int i = tid; i < plan.splits; i += DS_WG) m = fmaxf(m, part[2 * i]);
  const float M = block_max<DS_WAVES>(m, red);
  float s = 0.f;
  for (int i = tid; i < plan.splits; i += DS_WG) {
    const float mi = part[2 * i];
    s += mi == -INFINITY ? part[2 * i + 1] : part[2 * i + 1] * ds_rescale(mi, M, c, lo);
  }
  s = block_sum<DS_WAVES>(s, red);
  if (tid < 64) ds_finish<64>(a, plan, row, l.idx, l.v, l.z, [&](int i) { return l.first[i]; }, true, M, s, tid);
}

// ---- many short rows: TPR lanes of a wave a row, 8 columns each at a time; several rows a workgroup, none of which waits for another.
// A row's fixed work (what is listed, three 64-bit logarithms, the state) is as long as its columns': with a workgroup a row, 65536 x 100 fp32 took 468 us
// forward and 218 backward, with 16 lanes 23 and 11.  Pieces are laid out as in a row of channels: the last one is moved back to end with the row, what it repeats is left out.
template <int FMT, int TPR> struct DsShortRow {
  const typename RowElem<FMT>::type* z;
  int V, l;
  __device__ __forceinline__ int col(int i) const { return (i * TPR + l) * 8; }
  __device__ __forceinline__ int at(int i) const { return V < 8 ? 0 : min(col(i), V - 8); }
  __device__ __forceinline__ int rounds() const { return (V + TPR * 8 - 1) / (TPR * 8); }
  __device__ __forceinline__ RowRaw<FMT> load(int i) const { return load_piece<FMT>(z + at(i), min(V, 8), 0.f); }
};
__device__ __forceinline__ int ds_short_words(int V) { return V / 32 + 2; }         // (8 bits from any column on lie inside)
// (16 rows of 512 columns and 256 entries, 4 of 16384 and 256: at most 50 KB)
static size_t ds_short_lds(int V, int k, int sub, bool fwd) { return (size_t)4 * sub * (fwd ? V / 32 + 2 + 3 * k : 3 * k); }

template <int FMT, bool REST, int TPR> __global__ void __launch_bounds__(256) distill_short_fwd_kernel(rumpy_distill_args a, DsPlan plan) {
  typedef typename RowElem<FMT>::type E;
  extern __shared__ uint32_t bits_of_rows[];
  const int tid = threadIdx.x, lane = tid & 63, l = tid % TPR, words = ds_short_words(a.V);
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + tid / TPR;
  const bool in = row < a.rows, live = in && !(a.row_weight && a.row_weight[row] == 0.f);       // a row that does not count is not looked at
  if (in && !live && l == 0) { a.row_loss[row] = 0.f; a.state[row * DS_STATE + 5] = 1.f; }
  uint32_t* bits = bits_of_rows + (size_t)(tid / TPR) * (words + 3 * a.k);
  int* idx = reinterpret_cast<int*>(bits + words);
  float* v = reinterpret_cast<float*>(idx + a.k);
  float* zl = v + a.k;
  const DsShortRow<FMT, TPR> r{reinterpret_cast<const E*>(a.logits) + (size_t)(live ? row : 0) * a.ld, a.V, l};
  RowRaw<FMT> raw;
  if (live) raw = r.load(0);
  for (int i = l; i < words; i += TPR) bits[i] = 0;
  __syncthreads();
  bool twice = false;
  if (live) {
    for (int i = l; i < a.k; i += TPR) {
      const int64_t j = ds_index(a, row, i);
      const bool inside = j >= 0 && j < a.V;
      idx[i] = j < 0 ? -1 : inside ? (int)j : -2;
      v[i] = ds_value(a, row, i);
      zl[i] = inside ? elem_to_f32<FMT>(r.z[j]) : 0.f;
      if (inside) twice |= atomicOr(&bits[j >> 5], 1u << (j & 31)) >> (j & 31) & 1u;
    }
  }
  __syncthreads();
  if (!live) return;
  const float c = plan.c, lo = plan.lo;
  float m = -INFINITY, ref = 0.f, s = 0.f;
  const int rounds = r.rounds();
  for (int b = 0; b < rounds; ++b) {
    float x[8];
    unpack_piece<FMT>(raw, x);
    if (b + 1 < rounds) raw = r.load(b + 1);
    const int col = r.col(b), at = r.at(b);
    uint32_t out = 0;
    if constexpr (REST) {
      const uint32_t* w = bits + (at >> 5);
      out = (uint32_t)((((uint64_t)w[1] << 32) | w[0]) >> (at & 31));
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if ((out >> i & 1u) || at + i < col || at + i >= a.V) x[i] = -INFINITY;
      top = fmaxf(top, x[i]);
    }
    if (top > m) {
      s *= ds_rescale(m, top, c, lo);
      m = ref = top;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s += ds_exp(x[i], ref, c, lo);
  }
  const float M = lanes_max<TPR>(m, lane);
  s = lanes_sum<TPR>(m == -INFINITY ? s : s * ds_rescale(m, M, c, lo), lane);
  const bool doubled = lanes_any<TPR>(twice, lane);
  // (the row's columns are looked through only where one is named twice)
  auto first = [&](int i) {
    if (doubled)
      for (int o = 0; o < i; ++o) if (idx[o] == idx[i]) return false;
    return true;
  };
  ds_finish<TPR>(a, plan, row, idx, v, zl, first, doubled, M, s, lane);
}

// loss = sum of the rows' (weighted) losses, over the sum of the weights for the mean; a sum of weights of zero gives 0
// (one workgroup: 8 rows a thread are asked for together)
__global__ void __launch_bounds__(1024) distill_total_kernel(rumpy_distill_args a) {
  __shared__ double red[2][16];
  double s = 0.0, w = 0.0;
  for (int64_t r0 = threadIdx.x; r0 < a.rows; r0 += 8 * 1024) {
    float l[8], wr[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + i * 1024;
      l[i] = r < a.rows ? a.row_loss[r] : 0.f;
      wr[i] = r >= a.rows ? 0.f : a.row_weight ? a.row_weight[r] : 1.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) { s += l[i]; w += wr[i]; }
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) { s += __shfl_xor(s, o); w += __shfl_xor(w, o); }
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = s; red[1][threadIdx.x >> 6] = w; }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = w = 0.0;
    for (int i = 0; i < 16; ++i) { s += red[0][i]; w += red[1][i]; }
    const double f = !a.mean ? 1.0 : w == 0.0 ? 0.0 : 1.0 / w;
    *a.factor = (float)f;
    *a.loss = f == 0.0 ? 0.f : (float)(s * f);
  }
}

// The gradient: one exponential per column on the way through (4096 x 50021 bf16: 154 us = 5.3 TB/s read + written), then the row's few listed columns.
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
  const float c = plan.near;               // (the row's stream)
  float g = (a.loss ? *a.gout * *a.factor : a.gout[row]) * (float)a.tau;
  if (a.row_weight) g *= a.row_weight[row];
  const float m = st[0], coef = g * st[1];
  if (tid < a.k) {
    const int64_t i = ds_index(a, row, tid);
    idx[tid] = i >= j0 && i < j1 ? (int)i : -1;
    p[tid] = i < 0 ? 0.f : ds_exp(ds_value(a, row, tid), st[6], plan.c, plan.lo) * st[4];
  }
  for (int64_t j = j0 + tid * 8; j < j1; j += DS_WG * 8) {
    const int n = (int)min((int64_t)8, j1 - j);
    float v[8];
    unpack_piece<FMT>(load_piece<FMT>(z + j, n, 0.f), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = coef * __builtin_amdgcn_exp2f((v[i] - m) * c);
    store8<FMT>(a.dlogits, out + j, n, v);
  }
  __syncthreads();          // the listed columns are written over (same workgroup, behind the barrier); a column listed twice takes both shares
  if (tid < a.k && idx[tid] >= 0) {
    float share = 0.f;
    const int mine = idx[tid];
    for (int o = 0; o < a.k; o += 16) {
      int other[16];
      float po[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) { other[i] = idx[o + i]; po[i] = p[o + i]; }
#pragma unroll
      for (int i = 0; i < 16; ++i) share += o + i < a.k && other[i] == mine ? po[i] : 0.f;
    }
    const float q = ds_exp(elem_to_f32<FMT>(z[idx[tid]]), st[2], plan.c, plan.lo) * st[3];
    reinterpret_cast<E*>(a.dlogits)[out + idx[tid]] = f32_to_elem<FMT>(g * (q - share));
  }
}

// many short rows, as in the forward pass: the listed columns' gradients are made first and stored over the others'
template <int FMT, int TPR> __global__ void __launch_bounds__(256) distill_short_bwd_kernel(rumpy_distill_args a, DsPlan plan) {
  typedef typename RowElem<FMT>::type E;
  extern __shared__ uint32_t listed_of_rows[];
  const int tid = threadIdx.x, l = tid % TPR;
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + tid / TPR;
  const bool in = row < a.rows;
  int* idx = reinterpret_cast<int*>(listed_of_rows + (size_t)(tid / TPR) * 3 * a.k);
  float* p = reinterpret_cast<float*>(idx + a.k);
  float* q = p + a.k;
  const DsShortRow<FMT, TPR> r{reinterpret_cast<const E*>(a.logits) + (size_t)(in ? row : 0) * a.ld, a.V, l};
  const float* st = a.state + (in ? row : 0) * DS_STATE;
  const bool live = in && st[5] == 0.f, doubled = st[7] != 0.f;
  const float c = plan.near;
  float g = 0.f;
  E* out = reinterpret_cast<E*>(a.dlogits) + (size_t)(in ? row : 0) * a.V;
  if (live) {
    g = (a.loss ? *a.gout * *a.factor : a.gout[row]) * (float)a.tau;
    if (a.row_weight) g *= a.row_weight[row];
    for (int i = l; i < a.k; i += TPR) {
      const int64_t j = ds_index(a, row, i);
      const bool inside = j >= 0 && j < a.V;
      idx[i] = inside ? (int)j : -1;
      p[i] = j < 0 ? 0.f : ds_exp(ds_value(a, row, i), st[6], plan.c, plan.lo) * st[4];
      q[i] = inside ? ds_exp(elem_to_f32<FMT>(r.z[j]), st[2], plan.c, plan.lo) * st[3] : 0.f;
    }
  }
  if (in) {
    const float m = live ? st[0] : 0.f, coef = live ? g * st[1] : 0.f;
    for (int b = 0; b < r.rounds(); ++b) {
      if (r.col(b) >= a.V) break;
      float x[8];
      if (live) unpack_piece<FMT>(r.load(b), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = live ? coef * __builtin_amdgcn_exp2f((x[i] - m) * c) : 0.f;
      store8<FMT>(out, r.at(b), min(a.V, 8), x);
    }
  }
  __syncthreads();
  if (!live) return;
  for (int i = l; i < a.k; i += TPR) {
    const int mine = idx[i];
    if (mine < 0) continue;
    float share = p[i];
    if (doubled) {
      share = 0.f;
      for (int o = 0; o < a.k; ++o) share += idx[o] == mine ? p[o] : 0.f;
    }
    out[mine] = f32_to_elem<FMT>(g * (q[i] - share));
  }
}

static bool ds_fmt(int f) { return f == RUMPY_FMT_F32 || f == RUMPY_FMT_BF16 || f == RUMPY_FMT_F16; }
static const char* ds_check(const rumpy_distill_args* p) {
  if (!p) return "no arguments";
  if (!ds_fmt(p->fmt) || !ds_fmt(p->value_fmt)) return "fp32, bf16 or fp16 logits and top logits";
  if (p->rows < 0 || p->V < 1 || p->V > DS_MAXV || p->ld < 0) return "rows of 1 .. 2^30 logits";
  if (p->k < 1 || p->k > DS_MAXK) return "1 .. 256 top logits a row";
  if (!(p->tau >= 1e-30 && p->tau <= 1e30)) return "a temperature above zero";
  if (p->rows && (!p->logits || !p->top_values || !p->top_indices || !p->row_loss || !p->state)) return "a tensor is missing";
  if (p->loss && !p->factor) return "the reduction's factor is missing";
  if (p->rows > 0x7fffffff) return "at most 2^31 - 1 rows";
  const DsPlan plan = ds_plan(p->rows, p->V, p->tau);
  if (plan.splits > 1 && !p->partial) return "rows of this length and number are cut and need `partial` (rumpy_distill_partial_floats)";
  return nullptr;
}
extern "C" int64_t rumpy_distill_partial_floats(int64_t rows, int32_t V) {
  if (rows <= 0 || V < 1 || V > DS_MAXV) return 0;
  const DsPlan plan = ds_plan(rows, V, 1.0);
  return plan.splits > 1 ? rows * plan.splits * 2 : 0;
}

// Lanes of a short row; 0: a workgroup a row, or more.  us, bf16, forward + gradient, 16 lanes | 64 lanes | a workgroup a row:
//   65536 x 100, k 8: 23 + 11 | 87 + 29 | 468 + 218     4096 x 256, k 64: 11 + 7 | 10 + 5 | 40 + 13     300 x 1000, k 8: 11 + 6 | 7 + 4 | 8 + 4
//   16384 x 1000, k 8: 18 + 14 | 30 + 15 | 113 + 45      1200 x 2000, k 8: 9 + 6 (64) | 14 + 6      300 x 4000, k 8: 11 + 7 (64) | 7 + 4
//   4096 x 4000, k 64: 18 + 14 (64) | 43 + 18            4096 x 8192, k 8: 24 + 24 (64) | 35 + 23     1200 x 8000, k 8: 19 + 13 (64) | 14 + 9
//   8192 x 12001, k 8: 54 + 83 (64) | 91 + 75            2048 x 16000, k 8: 28 + 25 (64) | 24 + 22
// So 16 lanes while a row's columns and entries are few a lane and there are rows for all lanes of the chip; 64 while the rows fill it with a wave each
// (the gradient, which streams more and has less to do for a row, up to 4096 columns).
static int ds_short(int64_t rows, int32_t V, int32_t k, bool fwd) {
  if (rows >= 8192 ? V <= (k <= 32 ? 1024 : 512) : V <= 256 && k <= 16) return 16;
  if (V <= 1024) return 64;
  return rows * 4 >= V && V <= (!fwd ? 4096 : rows >= 4096 ? 16384 : 8192) ? 64 : 0;
}
static rumpy_distill_args ds_part(const rumpy_distill_args& a, const DsPlan& plan, int64_t r, int64_t n) {
  rumpy_distill_args b = a;
  b.rows = n;
  advance(b.logits, r * a.ld * elem_bytes(a.fmt)); advance(b.top_values, r * a.k * elem_bytes(a.value_fmt)); advance(b.top_indices, r * a.k * (a.index64 ? 8 : 4));
  advance(b.tail, r * 4); advance(b.row_weight, r * 4); advance(b.row_loss, r * 4); advance(b.state, r * DS_STATE * 4);
  advance(b.dlogits, r * a.V * elem_bytes(a.fmt));
  if (plan.splits > 1) advance(b.partial, r * plan.splits * 8);
  if (!a.loss) advance(b.gout, r * 4);
  return b;
}
template <int FMT, int TPR> static void ds_launch_short_fwd(const rumpy_distill_args& a, const DsPlan& plan, hipStream_t s) {
  constexpr int SUB = 256 / TPR;
  const dim3 grid((unsigned)((a.rows + SUB - 1) / SUB));
  const size_t lds = ds_short_lds(a.V, a.k, SUB, true);
  if (a.tail) hipLaunchKernelGGL((distill_short_fwd_kernel<FMT, true, TPR>), grid, dim3(256), lds, s, a, plan);
  else hipLaunchKernelGGL((distill_short_fwd_kernel<FMT, false, TPR>), grid, dim3(256), lds, s, a, plan);
}
template <int FMT> static void ds_launch_bwd(const rumpy_distill_args& all, const DsPlan& plan, hipStream_t s) {
  const int tpr = ds_short(all.rows, all.V, all.k, false);
  const size_t lds = tpr ? ds_short_lds(all.V, all.k, 256 / tpr, false) : 0;
  rows_in_parts(all.rows, tpr ? tpr : (int64_t)DS_WG * plan.splits, [&](int64_t r, int64_t n) {
    const rumpy_distill_args a = ds_part(all, plan, r, n);
    if (tpr == 16) hipLaunchKernelGGL((distill_short_bwd_kernel<FMT, 16>), dim3((unsigned)((n + 15) / 16)), dim3(256), lds, s, a, plan);
    else if (tpr == 64) hipLaunchKernelGGL((distill_short_bwd_kernel<FMT, 64>), dim3((unsigned)((n + 3) / 4)), dim3(256), lds, s, a, plan);
    else hipLaunchKernelGGL((distill_bwd_kernel<FMT>), dim3((unsigned)(n * plan.splits)), dim3(DS_WG), 0, s, a, plan);
  });
}
template <int FMT> static void ds_launch_fwd(const rumpy_distill_args& all, const DsPlan& plan, hipStream_t s) {
  const int tpr = ds_short(all.rows, all.V, all.k, true);
  rows_in_parts(all.rows, tpr ? tpr : (int64_t)DS_WG * plan.splits, [&](int64_t r, int64_t n) {
    const rumpy_distill_args a = ds_part(all, plan, r, n);
    if (tpr == 16) return ds_launch_short_fwd<FMT, 16>(a, plan, s);
    if (tpr == 64) return ds_launch_short_fwd<FMT, 64>(a, plan, s);
    const dim3 grid((unsigned)(n * plan.splits));
    const size_t lds = a.tail ? ((size_t)(plan.splits == 1 ? a.V : plan.seg) + 7 + 31) / 32 * 4 : 0;
    if (a.tail) hipLaunchKernelGGL((distill_fwd_kernel<FMT, true>), grid, dim3(DS_WG), lds, s, a, plan);
    else hipLaunchKernelGGL((distill_fwd_kernel<FMT, false>), grid, dim3(DS_WG), 0, s, a, plan);
    if (plan.splits > 1) hipLaunchKernelGGL((distill_join_kernel<FMT>), dim3((unsigned)n), dim3(DS_WG), 0, s, a, plan);
  });
}
extern "C" int rumpy_distill_fwd(const rumpy_distill_args* p, void* stream) {
  const char* bad = ds_check(p);
  if (bad) { rumpy_set_error("rumpy_distill_fwd: %s", bad); return RUMPY_E_ARG; }
  hipStream_t s = (hipStream_t)stream;
  if (p->rows) {
    const DsPlan plan = ds_plan(p->rows, p->V, p->tau);
    if (p->fmt == RUMPY_FMT_F32) ds_launch_fwd<RUMPY_FMT_F32>(*p, plan, s);
    else if (p->fmt == RUMPY_FMT_BF16) ds_launch_fwd<RUMPY_FMT_BF16>(*p, plan, s);
    else ds_launch_fwd<RUMPY_FMT_F16>(*p, plan, s);
  }
  if (p->loss) hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(1024), 0, s, *p);
  return rumpy_check_launch("rumpy_distill_fwd");
}
extern "C" int rumpy_distill_bwd(const rumpy_distill_args* p, void* stream) {
  const char* bad = ds_check(p);
  if (!bad && p->rows && (!p->dlogits || !p->gout)) bad = "a tensor is missing";
  if (bad) { rumpy_set_error("rumpy_distill_bwd: %s", bad); return RUMPY_E_ARG; }
  if (p->rows == 0) return RUMPY_OK;
  const DsPlan plan = ds_plan(p->rows, p->V, p->tau);
  hipStream_t s = (hipStream_t)stream;
  if (p->fmt == RUMPY_FMT_F32) ds_launch_bwd<RUMPY_FMT_F32>(*p, plan, s);
  else if (p->fmt == RUMPY_FMT_BF16) ds_launch_bwd<RUMPY_FMT_BF16>(*p, plan, s);
  else ds_launch_bwd<RUMPY_FMT_F16>(*p, plan, s);
  return rumpy_check_launch("rumpy_distill_bwd");
}
