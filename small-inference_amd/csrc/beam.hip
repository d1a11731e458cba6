// Beams: the best continuations over the beams and the vocabulary of a request, and the copies of blocks of beams that go on
// from the same one (gfx950). The reference decodes greedily and has no counterpart.
//
// Selection, for row r (a beam) and token v:  score = cum[r] + l[r, v] - log sum_v exp(l[r, v]).  Within a row the logits
// decide the order, so that one pass over them finds a row's best tokens and its sum together:
//   beam_rows   a workgroup holds a piece of a row in registers, takes its maximum, the sum of exponentials below it, and
//               its N largest logits: those above a threshold that at least N pass (the N-th largest of the threads' maxima)
//               are collected in LDS and put into order by counting.
//   beam_merge  a workgroup a group, a wave a row: joins the pieces' sums in 64 bits and puts a row's candidates, then the
//               group's, in order in the same way.
// 512 rows of 151936 bf16 logits, 16 candidates of 8 rows each: 37.5 us and 6.5 (30.6 as a copy's rate reads them), bound by
// memory and the exponentials' vector operations in turn; a few rows by the round trips of both kernels, 5 and 6 us.
// It reads every logit once; no sum depends on the order in which workgroups or waves run, so equal rows get equal sums.
// A row's log-sum is within 2^-19: of its terms exp(-d), d the distance to the piece's largest logit, an exponent's argument is
// off by d 2^-22.8 at most (difference, constant and product rounded), exp2 by 2^-23, the sum of eight by 7 2^-24; the mean of d
// over a piece's weights is under 6.8 whatever the piece's 16384 logits are (one on top, the others W(16384 / e) below it).
#include <algorithm>
#include <memory>
#include <new>

#include "decode_common.h"

namespace sipa {

constexpr int kBeamThreads = 256, kBeamMaxN = 64, kBeamMaxRows = 1024;
constexpr int kBeamCap = 256;  // collected logits of a wave

struct BeamArgs {
  const void* logits;
  int64_t l_st;
  const float* cum;
  const int32_t* starts;
  int32_t R, V, beams, N;
  int32_t ns, piece;  // pieces of a row, logits of a piece
  float* p_max;       // [R][ns]
  double* p_sum;      // [R][ns] sum of exp(l - p_max)
  uint64_t* p_key;    // [R][N][ns] the pieces' largest logits in order (beam_key), 0 behind them
  float* out_scores;
  int64_t* out_beams;
  int64_t* out_tokens;
};

// fp32 as an integer of the same order; of equal values the lower index is the larger key. No value but NaN gives 0.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as 0
  return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~index;
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// fp64 as an integer of the same order, 0 for none.
__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.);
  return b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ double score_value(uint64_t b) {
  return __builtin_bit_cast(double, b >> 63 ? b & ~(1ull << 63) : ~b);
}

// Step K = 0 .. 5 of a butterfly over a wave: the value of a lane that the steps before have not brought together with this one.
// Cross-lane moves of the vector unit, without LDS.
template <int K>
__device__ __forceinline__ uint32_t other_lane(uint32_t x) {
  if constexpr (K == 0) {
    const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? p[0] : p[1];
  } else if constexpr (K == 1) {
    const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? p[0] : p[1];
  }
  else if constexpr (K == 2) return __builtin_amdgcn_update_dpp(x, x, 0x128, 0xf, 0xf, true);  // 8 further of 16
  else if constexpr (K == 3) return __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, true);  // 7 - i of 8
  else if constexpr (K == 4) return __builtin_amdgcn_update_dpp(x, x, 0x4E, 0xf, 0xf, true);   // 2 3 0 1 of 4
  else return __builtin_amdgcn_update_dpp(x, x, 0xB1, 0xf, 0xf, true);                         // 1 0 3 2
}

template <int K>
__device__ __forceinline__ float other_lane(float x) {
  return __uint_as_float(other_lane<K>(__float_as_uint(x)));
}

template <int K>
__device__ __forceinline__ uint64_t other_lane(uint64_t x) {
  return (uint64_t)other_lane<K>((uint32_t)(x >> 32)) << 32 | other_lane<K>((uint32_t)x);
}

template <int K>
__device__ __forceinline__ double other_lane(double x) {
  return __builtin_bit_cast(double, other_lane<K>(__builtin_bit_cast(uint64_t, x)));
}

template <int K = 0, typename T, typename F>
__device__ __forceinline__ T butterfly(T x, F f) {  // f(K, own, other); every lane gets the result
  if constexpr (K == 6) return x;
  else return butterfly<K + 1>(f(K, x, other_lane<K>(x)), f);
}

// fp32's upper 16 bits in order, and the least value that has them.
__device__ __forceinline__ uint32_t upper_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> 16;
}

__device__ __forceinline__ float upper_value(uint32_t key) {
  return __uint_as_float(key & 0x8000u ? (key & 0x7fffu) << 16 : ~(key << 16));
}

// The N-th largest of a wave's 64 C 16-bit keys, C a lane (0 if there are fewer): a bit at a time, by counting.
template <int C>
__device__ __forceinline__ uint32_t nth_key(const uint32_t (&key)[C], int N) {
  uint32_t t = 0;
#pragma unroll
  for (uint32_t bit = 0x8000u; bit > 0; bit >>= 1) {
    int over = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) over += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] >= (t | bit)));
    t = over >= N ? t | bit : t;
  }
  return t;
}

__device__ __forceinline__ double wave_sum_f64(double x) {  // a + b and b + a are the same bits
  return butterfly(x, [](int, double a, double b) { return a + b; });
}

// How many of the keys of a list in LDS (in fours, with 0 behind the last) are over `key`.
__device__ __forceinline__ int keys_over(const uint64_t* list, int n, uint64_t key) {
  int over = 0;
#pragma unroll 1
  for (int j = 0; j < n; j += 4) {
    const ulonglong2 a = *(const ulonglong2*)(list + j), b = *(const ulonglong2*)(list + j + 2);
    over += (a.x > key) + (a.y > key) + (b.x > key) + (b.y > key);
  }
  return over;
}

__device__ __forceinline__ int keys_over(const uint32_t* list, int n, uint32_t key) {
  int over = 0;
#pragma unroll 1
  for (int j = 0; j < n; j += 4) {
    const uint4 a = *(const uint4*)(list + j);
    over += (a.x > key) + (a.y > key) + (a.z > key) + (a.w > key);
  }
  return over;
}

// A row's element: bits, how many make 16 bytes, and the key that orders those of a piece. Of 16-bit types it has 32 bits, the
// value's 16 and the place's within the piece: half the LDS reads and comparisons.
template <int DT>
struct BeamType {
  typedef uint16_t T;
  typedef uint32_t Key;
  static constexpr int E = 8;
  static __device__ __forceinline__ Key key(uint32_t bits, uint32_t at) {
    bits = bits == 0x8000u ? 0u : bits;  // -0 as 0
    return (bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u) << 16 | (0xffffu - at);
  }
  static __device__ __forceinline__ uint32_t bits(Key key) { return key >> 31 ? key >> 16 & 0x7fffu : ~(key >> 16) & 0xffffu; }
  static __device__ __forceinline__ uint32_t place(Key key) { return 0xffffu - (key & 0xffffu); }
};
template <>
struct BeamType<SIPA_F32> {
  typedef uint32_t T;
  typedef uint64_t Key;
  static constexpr int E = 4;
  static __device__ __forceinline__ Key key(uint32_t bits, uint32_t at) { return beam_key(__uint_as_float(bits), at); }
  static __device__ __forceinline__ uint32_t bits(Key key) { return __float_as_uint(key_value(key)); }
  static __device__ __forceinline__ uint32_t place(Key key) { return ~(uint32_t)key; }
};

template <int DT>
__device__ __forceinline__ float logit(uint32_t bits) {
  return DT == SIPA_F32 ? __uint_as_float(bits) : DT == SIPA_BF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32(bits);
}

// PARTS 16-byte parts of a row a thread (aligned to an element only: rows of an odd vocabulary start anywhere).
template <int DT, int PARTS>
__global__ void __launch_bounds__(kBeamThreads) beam_rows_kernel(const BeamArgs a) {
  typedef typename BeamType<DT>::T T;
  typedef typename BeamType<DT>::Key Key;
  constexpr int THR = kBeamThreads, E = BeamType<DT>::E, BITS = 8 * sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Part {
    uint32_t w[4];
  };
  __shared__ __align__(16) Key found[4][kBeamCap + 4];
  __shared__ float w_max[4][64];
  __shared__ double w_sum[4];
  __shared__ int w_count[4];
  __shared__ Key w_key[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x / a.ns, piece = blockIdx.x - r * a.ns, v0 = piece * a.piece;
  const T* row = (const T*)a.logits + (int64_t)r * a.l_st + v0;
  const int n = min(a.piece, a.V - v0);
  Part x[PARTS];
  constexpr uint32_t kNone = DT == SIPA_F32 ? 0xff800000u : DT == SIPA_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int at = E * (tid + THR * i);
    if (at + E <= n) x[i] = *(const Part*)(row + at);
    else x[i] = Part{{kNone, kNone, kNone, kNone}};
  }
  if (const int last = n / E; n % E != 0 && last % THR == tid) {  // the row's last few logits
    Part y = {{kNone, kNone, kNone, kNone}};
    for (int e = 0; e < n % E; ++e) {
      const uint32_t bits = row[last * E + e], shift = BITS * e & 31, mask = BITS == 32 ? ~0u : 0xffffu << shift;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (BITS * e >> 5 == w) y.w[w] = (y.w[w] & ~mask) | bits << shift;
    }
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
      if (last / THR == i) x[i] = y;
  }
  auto bits = [&](int i, int e) {
    const uint32_t w = x[i].w[BITS * e >> 5];
    return BITS == 32 ? w : e & 1 ? w >> 16 : w & 0xffffu;
  };
  auto value = [&](int i, int e) {
    const uint32_t w = x[i].w[BITS * e >> 5];
    if constexpr (DT == SIPA_BF16) return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    return logit<DT>(bits(i, e));
  };
  auto place = [&](int i, int e) { return (uint32_t)(E * (tid + THR * i) + e); };
  float mine = kNegInf;
#pragma unroll
  for (int i = 0; i < PARTS; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) mine = fmaxf(mine, value(i, e));
  // Kept as they came: the compiler would otherwise hold every logit in fp32, or its key (244 registers for 64 logits).
  auto keep = [&]() {
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) asm volatile("" : "+v"(x[i].w[w]));
  };
  keep();
  // Of the threads' maxima, or those of four threads each, the N-th largest is a threshold that N logits pass at least, and few
  // more do (N = 16: 18 of a piece of 16384; the least maximum of 16 classes of threads let 53 pass, whose collection took a
  // third of the time).
  w_max[wave][lane] = mine;
  __syncthreads();
  const float of[4] = {w_max[0][lane], w_max[1][lane], w_max[2][lane], w_max[3][lane]};
  const float best = fmaxf(fmaxf(of[0], of[1]), fmaxf(of[2], of[3]));
  const float top = butterfly(best, [](int, float p, float q) { return fmaxf(p, q); });
  float low;
  if (a.N <= 32) {
    const uint32_t key[1] = {upper_key(best)};
    low = upper_value(nth_key(key, a.N));
  } else {
    const uint32_t key[4] = {upper_key(of[0]), upper_key(of[1]), upper_key(of[2]), upper_key(of[3])};
    low = upper_value(nth_key(key, a.N));
  }
  // exp(l - top) as exp2((l - top) log2 e), the argument rounded (the bound of the sum is at the top).
  const float off = top == kNegInf ? 0.f : top;
  low = fmaxf(low, -__FLT_MAX__);  // never -inf (or NaN, which the key 0 stands for)
  double sum = 0.;
  int count = 0;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = value(i, e);
      s += fast_exp2((v - off) * 1.44269504088896340736f);
      const uint64_t hits = __builtin_amdgcn_ballot_w64(v >= low);
      if (hits) {
        const int to = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0u));
        if (v >= low && to < kBeamCap) found[wave][to] = BeamType<DT>::key(bits(i, e), place(i, e));
        count += __builtin_popcountll(hits);
      }
    }
    sum += (double)s;
  }
  sum = wave_sum_f64(sum);
  if (lane < 4 && count <= kBeamCap) found[wave][count + lane] = 0;
  if (lane == 0) w_sum[wave] = sum, w_count[wave] = count;
  __syncthreads();
  const int64_t at = (int64_t)r * a.ns + piece;
  if (tid == 0) {
    a.p_max[at] = top;
    a.p_sum[at] = (w_sum[0] + w_sum[1]) + (w_sum[2] + w_sum[3]);
  }
  auto store = [&](int rank, Key key) {
    a.p_key[((int64_t)r * a.N + rank) * a.ns + piece] =
        beam_key(logit<DT>(BeamType<DT>::bits(key)), (uint32_t)v0 + BeamType<DT>::place(key));
  };
  const int all[4] = {w_count[0], w_count[1], w_count[2], w_count[3]};
  int got = 0;
  if (max(max(all[0], all[1]), max(all[2], all[3])) <= kBeamCap) {
    got = all[0] + all[1] + all[2] + all[3];
    for (int i = lane; i < count; i += 64) {
      const Key key = found[wave][i];  // no two are equal
      int rank = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) rank += keys_over(found[w], all[w], key);
      if (rank < a.N) store(rank, key);
    }
  } else {
    // Most of the piece ties or rises: the largest key under the last one, N times. Only the thread that had it looks for
    // its next.
    auto best_below = [&](Key limit) {
      Key best = 0;
#pragma unroll 1
      for (int i = 0; i < PARTS; ++i)
#pragma unroll 1
        for (int e = 0; e < E && (int)place(i, e) < n; ++e) {
          const uint32_t b = row[place(i, e)];
          const Key key = logit<DT>(b) > kNegInf ? BeamType<DT>::key(b, place(i, e)) : 0;
          best = key < limit && key > best ? key : best;
        }
      return best;
    };
    Key own = best_below(~(Key)0);
    for (; got < a.N; ++got) {
      Key best = butterfly(own, [](int, Key p, Key q) { return p > q ? p : q; });
      if (lane == 0) w_key[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w) best = w_key[w] > best ? w_key[w] : best;
      __syncthreads();
      if (best == 0) break;  // uniform
      if (own == best) {
        store(got, best);
        own = best_below(best);
      }
    }
  }
  for (int i = got + tid; i < a.N; i += THR) a.p_key[((int64_t)r * a.N + i) * a.ns + piece] = 0;
}

// The N largest of a wave's keys (no two equal, 0: none), SLOTS a lane, in order, to best[0 ..] in LDS. list: room for
// 64 SLOTS + 4 keys.
template <int SLOTS>
__device__ __forceinline__ void wave_select(const uint64_t (&key)[SLOTS], int N, uint64_t* list, uint64_t* best) {
  const int lane = threadIdx.x & 63;
  uint64_t most = 0;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) most = key[i] > most ? key[i] : most;
  const uint32_t upper[1] = {(uint32_t)(most >> 48)};
  const uint64_t low = max((uint64_t)nth_key(upper, N) << 48, (uint64_t)1);
  int n = 0;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const uint64_t hits = __builtin_amdgcn_ballot_w64(key[i] >= low);
    if (hits) {
      const int to = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0u));
      if (key[i] >= low) list[to] = key[i];
      n += __builtin_popcountll(hits);
    }
  }
  if (lane < 4) list[n + lane] = 0;
  wave_sync();
  for (int i = lane; i < n; i += 64) {
    const int rank = keys_over(list, n, list[i]);
    if (rank < N) best[rank] = list[i];
  }
}

constexpr int kMergeWaves = 8, kMergeSlots = 8;

// Eight rows at a time: each wave finds its row's candidates among those of the row's pieces, then where they stand among the
// other rows' and the group's so far (lists in order, searched by halving; of equal scores the earlier row's go first).
__global__ void __launch_bounds__(64 * kMergeWaves) beam_merge_kernel(const BeamArgs a) {
  constexpr int W = kMergeWaves, SLOTS = kMergeSlots + 1;
  __shared__ __align__(16) uint64_t list[W][64 * SLOTS + 4];
  __shared__ uint64_t row_best[W][kBeamMaxN];             // a row's candidates in order (beam_key)
  __shared__ uint64_t score[2][W + 1][kBeamMaxN];         // in turn: the group's so far, then the rows' (score_key)
  __shared__ uint64_t from[2][kBeamMaxN];                 // the group's so far: row << 32 | token
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = blockIdx.x, N = a.N;
  const int r0 = a.starts == nullptr ? g * a.beams : min(max(a.starts[g], 0), a.R);
  const int r1 = a.starts == nullptr ? r0 + a.beams : min(max(a.starts[g + 1], r0), a.R);
  const int rows = min(r1 - r0, kBeamMaxRows);
  if (wave == 0) score[0][0][lane] = 0;
  int turn = 0;
  for (int b0 = 0; b0 < rows; b0 += W, turn ^= 1) {
    const int b = b0 + wave;
    uint64_t mine = 0;  // lane i: the row's candidate i
    double off = __builtin_nan("");
    if (b < rows) {
      const int64_t first = (int64_t)(r0 + b) * a.ns;
      const uint64_t* keys = a.p_key + first * N;
      const int total = a.ns * N;
      uint64_t key[SLOTS];
      auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < kMergeSlots; ++i) key[i + 1] = keys[min(i0 + 64 * i + lane, total - 1)];
      };
      load(0);
      // the row's sum
      float m = lane < a.ns ? a.p_max[first + lane] : kNegInf, top = m;
      double s = lane < a.ns ? a.p_sum[first + lane] : 0.;
      for (int i = lane + 64; i < a.ns; i += 64) top = fmaxf(top, a.p_max[first + i]);
      top = butterfly(top, [](int, float p, float q) { return fmaxf(p, q); });
      double sum = 0.;
      for (int i = lane;;) {
        sum += m == kNegInf ? s : s * exp((double)m - (double)top);
        if ((i += 64) >= a.ns) break;
        m = a.p_max[first + i], s = a.p_sum[first + i];
      }
      sum = wave_sum_f64(sum);
      off = (double)a.cum[r0 + b] - ((double)top + log(sum));
      for (int i0 = 0; i0 < total; i0 += 64 * kMergeSlots) {
        if (i0 > 0) load(i0);
        key[0] = mine;
#pragma unroll
        for (int i = 0; i < kMergeSlots; ++i)
          if (i0 + 64 * i + lane >= total) key[i + 1] = 0;
        row_best[wave][lane] = 0;
        wave_sync();
        wave_select<SLOTS>(key, N, list[wave], row_best[wave]);
        wave_sync();
        mine = row_best[wave][lane];
      }
    }
    const bool live = fabs(off) < __builtin_huge_val();  // else no candidate is the row's
    const uint64_t own = mine != 0 && live ? score_key(off + (double)key_value(mine)) : 0;
    score[turn][wave + 1][lane] = own;
    if (wave == 0) score[turn ^ 1][0][lane] = 0;
    __syncthreads();
    auto place = [&](int of, uint64_t k) {  // candidates before the lane's: of earlier lists those not under it, of later ones those over it
      int at[W + 1];
#pragma unroll
      for (int w = 0; w <= W; ++w) at[w] = 0;
#pragma unroll
      for (int step = 32; step > 0; step >>= 1)
#pragma unroll
        for (int w = 0; w <= W; ++w) {
          const uint64_t x = score[turn][w][at[w] + step - 1];
          at[w] += x > k || (x == k && w < of) ? step : 0;
        }
      int sum = 0;
#pragma unroll
      for (int w = 0; w <= W; ++w) {  // (63 of the 64 places so far)
        const uint64_t x = score[turn][w][at[w]];
        sum += w == of ? 0 : at[w] + (x > k || (x == k && w < of));
      }
      return sum;
    };
    if (own != 0) {
      const int at = place(wave + 1, own) + lane;
      if (at < N) {
        score[turn ^ 1][0][at] = own;
        from[turn ^ 1][at] = (uint64_t)b << 32 | (uint32_t)~(uint32_t)mine;
      }
    }
    if (wave == W - 1 && b0 > 0 && score[turn][0][lane] != 0) {
      const int at = place(0, score[turn][0][lane]) + lane;
      if (at < N) {
        score[turn ^ 1][0][at] = score[turn][0][lane];
        from[turn ^ 1][at] = from[turn][lane];
      }
    }
    __syncthreads();
  }
  __syncthreads();
  if (wave == 0 && lane < N) {
    const uint64_t k = score[turn][0][lane], of = from[turn][lane];
    a.out_scores[(int64_t)g * N + lane] = k != 0 ? (float)score_value(k) : kNegInf;
    a.out_beams[(int64_t)g * N + lane] = k != 0 ? (int64_t)(of >> 32) : -1;
    a.out_tokens[(int64_t)g * N + lane] = k != 0 ? (int64_t)(uint32_t)of : -1;
  }
}

// ---- copies of blocks --------------------------------------------------------------------------------------------------

constexpr int kCopiesPerLaunch = 424, kCopyPools = 4, kCopyUnroll = 8;  // (as many as kernel arguments hold, 4 KB)

struct CopyArgs {
  char* pool[kCopyPools];
  int64_t st_l[kCopyPools], st_h[kCopyPools];
  int32_t row[kCopyPools];         // bytes of a token
  int32_t unit[kCopyPools];        // bytes moved at a time
  int32_t log_lanes[kCopyPools];   // lanes of a (layer, head)
  int32_t L, H, B;
  int32_t src[kCopiesPerLaunch], dst[kCopiesPerLaunch];
  uint8_t tokens[kCopiesPerLaunch];
};
static_assert(sizeof(CopyArgs) <= 4096, "kernel arguments");

// Workgroup (copy, y, pool): (layer, head) segments of one block, 1 << log_lanes lanes side by side on each, kCopyUnroll segments
// a thread with all their loads ahead of the stores, which go past the caches: 384 copies in 28 layers of INT8 pools, 128 MB read
// and written, 24 us (5.2 TB/s; with ordinary stores 41, with loads past the caches too 28).
template <typename U>
__device__ __forceinline__ void copy_segments(const CopyArgs& a, int pool, int c) {
  const int log_lanes = a.log_lanes[pool], per = 256 >> log_lanes, lane = threadIdx.x & ((1 << log_lanes) - 1);
  const int row = a.row[pool], units = a.tokens[c] * row / (int)sizeof(U), all = a.L * a.H;
  const int64_t block = (int64_t)a.B * row, to = (a.dst[c] - a.src[c]) * block, st_l = a.st_l[pool], st_h = a.st_h[pool];
  const int first = blockIdx.y * per * kCopyUnroll + (threadIdx.x >> log_lanes);
  if (first >= all || lane >= units) return;
  const int dl = per / a.H, dh = per - dl * a.H;  // uniform
  const int64_t step = dl * st_l + dh * st_h, wrap = st_l - a.H * st_h;
  const int l0 = first / a.H, h0 = first - l0 * a.H;
  char* base = a.pool[pool] + a.src[c] * block + l0 * st_l + h0 * st_h;
  for (int u = lane; u < units; u += 1 << log_lanes) {
    U x[kCopyUnroll];
    char* at = base + u * (int)sizeof(U);
    auto each = [&](auto f) {
      char* p = at;
      int h = h0;
#pragma unroll
      for (int i = 0; i < kCopyUnroll; ++i) {
        if (i == 0 || first + per * i < all) f(i, p);
        p += step;
        h += dh;
        p += h >= a.H ? wrap : 0;
        h -= h >= a.H ? a.H : 0;
      }
    };
    each([&](int i, char* p) { x[i] = *(const U*)p; });
    each([&](int i, char* p) { __builtin_nontemporal_store(x[i], (U*)(p + to)); });
  }
}

__global__ void __launch_bounds__(256) copy_blocks_kernel(const CopyArgs a) {
  const int pool = blockIdx.z, c = blockIdx.x;
  if (a.unit[pool] == 16) copy_segments<u32x4>(a, pool, c);
  else if (a.unit[pool] == 2) copy_segments<uint16_t>(a, pool, c);
  else copy_segments<uint8_t>(a, pool, c);
}

}  // namespace sipa

using namespace sipa;

// Parts of a thread: the most, up to 8, that leave two workgroups a CU; 2 at least, from 32 candidates on 4, as the merge pays for
// each piece. Times in us with 2 / 4 / 8 parts, 16-bit logits of 151936 tokens: 4 rows, 8 candidates 10.8 / 11.6 / 12.4; 32 rows
// 13.5 / 13.2 / 14.4; 128 rows, 16 candidates 25.3 / 20.6 / 20.6; 512 rows 61 / 45 / 42.5; 1 row, 64 candidates 28 / 20.5 / 19.3.
// (16 parts, 137 registers: 512 rows 50.)
static int beam_parts(const sipa_beam_params* p) {
  const int piece = kBeamThreads * (p->dtype == SIPA_F32 ? 4 : 8);
  const auto workgroups = [&](int parts) { return (int64_t)p->num_rows * ((p->vocab + piece * parts - 1) / (piece * parts)); };
  return workgroups(8) >= 512 ? 8 : workgroups(4) >= 512 || p->num_candidates >= 32 ? 4 : 2;
}

struct BeamLayout {
  int parts, ns, piece;
  int64_t sum, key, total;
};

static int beam_layout(const sipa_beam_params* p, BeamLayout* l) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_beam_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_beam_params (%d bytes)", (int)sizeof(sipa_beam_params));
  SIPA_CHECK(p->num_rows >= 0 && p->num_groups >= 0 && p->vocab > 0 && p->vocab <= 1 << 25, SIPA_EINVAL,
             "%d rows, %d groups, vocabulary %d (up to 2^25)", p->num_rows, p->num_groups, p->vocab);
  SIPA_CHECK(p->num_candidates >= 1 && p->num_candidates <= kBeamMaxN, SIPA_EUNSUPPORTED, "%d candidates (1 .. %d)",
             p->num_candidates, kBeamMaxN);
  SIPA_CHECK(p->dtype == SIPA_F32 || p->dtype == SIPA_BF16 || p->dtype == SIPA_F16, SIPA_EUNSUPPORTED, "logits of type %d", p->dtype);
  l->parts = beam_parts(p);
  const int e = p->dtype == SIPA_F32 ? 4 : 8, most = kBeamThreads * e * l->parts;
  l->ns = (p->vocab + most - 1) / most;
  l->piece = ((p->vocab + l->ns - 1) / l->ns + e - 1) / e * e;  // alike, whole parts
  l->ns = (p->vocab + l->piece - 1) / l->piece;
  const int64_t pieces = (int64_t)p->num_rows * l->ns;
  SIPA_CHECK(pieces <= (int64_t)(0xffffffffu / kBeamThreads) && p->num_groups <= (int32_t)(0xffffffffu / (64 * kMergeWaves)),
             SIPA_EUNSUPPORTED, "%d rows of %d pieces, %d groups: a launch holds 2^32 threads", p->num_rows, l->ns, p->num_groups);
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  l->sum = up(pieces * 4);
  l->key = l->sum + up(pieces * 8);
  l->total = l->key + up(pieces * p->num_candidates * 8);
  return SIPA_OK;
}

extern "C" int64_t sipa_beam_workspace_bytes(const sipa_beam_params* p) {
  BeamLayout l;
  const int rc = beam_layout(p, &l);
  return rc != SIPA_OK ? rc : l.total;
}

template <int DT>
static void launch_beam_rows(int parts, unsigned grid, hipStream_t st, const BeamArgs& a) {
  if (parts == 8) hipLaunchKernelGGL((beam_rows_kernel<DT, 8>), dim3(grid), dim3(kBeamThreads), 0, st, a);
  else if (parts == 4) hipLaunchKernelGGL((beam_rows_kernel<DT, 4>), dim3(grid), dim3(kBeamThreads), 0, st, a);
  else hipLaunchKernelGGL((beam_rows_kernel<DT, 2>), dim3(grid), dim3(kBeamThreads), 0, st, a);
}

extern "C" int32_t sipa_beam_select(const sipa_beam_params* p, void* stream) {
  BeamLayout l;
  const int rc = beam_layout(p, &l);
  if (rc != SIPA_OK) return rc;
  if (p->num_groups == 0) return SIPA_OK;
  SIPA_CHECK(p->out_scores && p->out_beams && p->out_tokens && (p->num_rows == 0 || (p->logits && p->scores)), SIPA_EINVAL,
             "NULL pointer");
  SIPA_CHECK(p->starts != nullptr || (p->beams >= 1 && p->beams <= kBeamMaxRows &&
                                      (int64_t)p->beams * p->num_groups <= p->num_rows), SIPA_EINVAL,
             "%d groups of %d beams (up to %d) in %d rows", p->num_groups, p->beams, kBeamMaxRows, p->num_rows);
  SIPA_CHECK(l.total == 0 || (p->workspace != nullptr && ((uintptr_t)p->workspace & 255) == 0 && p->workspace_bytes >= l.total),
             SIPA_EWORKSPACE, "a 256-byte aligned workspace of %lld bytes is needed (have %lld)", (long long)l.total,
             (long long)p->workspace_bytes);
  BeamArgs a;
  a.logits = p->logits;
  a.l_st = p->logits_stride;
  a.cum = p->scores;
  a.starts = p->starts;
  a.R = p->num_rows;
  a.V = p->vocab;
  a.beams = p->beams;
  a.N = p->num_candidates;
  a.ns = l.ns;
  a.piece = l.piece;
  char* ws = (char*)p->workspace;
  a.p_max = (float*)ws;
  a.p_sum = (double*)(ws + l.sum);
  a.p_key = (uint64_t*)(ws + l.key);
  a.out_scores = p->out_scores;
  a.out_beams = p->out_beams;
  a.out_tokens = p->out_tokens;
  hipStream_t st = (hipStream_t)stream;
  if (p->num_rows > 0) {
    const unsigned grid = (unsigned)(p->num_rows * l.ns);
    if (p->dtype == SIPA_F32) launch_beam_rows<SIPA_F32>(l.parts, grid, st, a);
    else if (p->dtype == SIPA_BF16) launch_beam_rows<SIPA_BF16>(l.parts, grid, st, a);
    else launch_beam_rows<SIPA_F16>(l.parts, grid, st, a);
  }
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)p->num_groups), dim3(64 * kMergeWaves), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "beam selection launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}

extern "C" int32_t sipa_check_copies(const int32_t* copies, int32_t num_copies, int32_t num_blocks, int32_t block_size) {
  SIPA_CHECK(num_copies >= 0 && num_blocks >= 0 && block_size > 0, SIPA_EINVAL, "%d copies, %d blocks of %d tokens", num_copies,
             num_blocks, block_size);
  if (num_copies == 0) return SIPA_OK;
  SIPA_CHECK(copies != nullptr, SIPA_EINVAL, "NULL pointer");
  for (int i = 0; i < num_copies; ++i) {
    const int32_t* c = copies + 3 * (int64_t)i;
    SIPA_CHECK(c[0] >= 0 && c[0] < num_blocks && c[1] >= 0 && c[1] < num_blocks && c[2] >= 0 && c[2] <= block_size,
               SIPA_EINVAL, "copy %d: %d tokens of block %d to block %d (%d blocks of %d tokens)", i, c[2], c[0], c[1],
               num_blocks, block_size);
  }
  // The destinations in a hash table at most half full (block + 1, 0 for free), then the sources looked up in it.
  constexpr int kHere = 1024;
  uint32_t here[kHere];
  std::unique_ptr<uint32_t[]> more;
  uint32_t* table = here;
  int64_t size = kHere;
  while (size < 2 * (int64_t)num_copies) size *= 2;
  if (size > kHere) {
    more.reset(new (std::nothrow) uint32_t[size]);
    SIPA_CHECK(more != nullptr, SIPA_EINVAL, "no memory for %d copies", num_copies);
    table = more.get();
  }
  std::fill(table, table + size, 0u);
  const auto slot = [&](int32_t block) {  // of the block, or the free one where it would stand
    int64_t i = ((uint32_t)block * 2654435761u) & (size - 1);
    while (table[i] != 0 && table[i] != (uint32_t)block + 1) i = (i + 1) & (size - 1);
    return i;
  };
  for (int i = 0; i < num_copies; ++i) {
    const int32_t d = copies[3 * (int64_t)i + 1];
    const int64_t at = slot(d);
    SIPA_CHECK(table[at] == 0, SIPA_EINVAL, "block %d is the destination of two copies", d);
    table[at] = (uint32_t)d + 1;
  }
  for (int i = 0; i < num_copies; ++i)
    SIPA_CHECK(table[slot(copies[3 * (int64_t)i])] == 0, SIPA_EINVAL,
               "block %d is the destination of one copy and the source of another", copies[3 * (int64_t)i]);
  return SIPA_OK;
}

extern "C" int32_t sipa_copy_blocks(const sipa_copy_params* p, void* stream) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_copy_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_copy_params (%d bytes)", (int)sizeof(sipa_copy_params));
  SIPA_CHECK(p->num_layers >= 0 && p->num_kv_heads >= 0 && p->num_blocks >= 0 && p->block_size > 0 &&
                 p->num_copies >= 0 && p->num_pools >= 1 && p->num_pools <= kCopyPools &&
                 (int64_t)p->num_layers * p->num_kv_heads <= 1 << 24, SIPA_EINVAL,
             "%d layers of %d heads, %d blocks of %d tokens, %d pools, %d copies", p->num_layers, p->num_kv_heads, p->num_blocks,
             p->block_size, p->num_pools, p->num_copies);
  if (p->num_copies == 0 || p->num_layers == 0 || p->num_kv_heads == 0) return SIPA_OK;
  SIPA_CHECK(p->block_size <= 255, SIPA_EUNSUPPORTED, "blocks of %d tokens (up to 255)", p->block_size);
  const int rc = sipa_check_copies(p->copies, p->num_copies, p->num_blocks, p->block_size);
  if (rc != SIPA_OK) return rc;
  CopyArgs a;
  a.L = p->num_layers;
  a.H = p->num_kv_heads;
  a.B = p->block_size;
  int most = 1;
  for (int i = 0; i < p->num_pools; ++i) {
    const int64_t row = p->row_bytes[i], of = (int64_t)(uintptr_t)p->pools[i] | p->stride_l[i] | p->stride_h[i] | row;
    SIPA_CHECK(p->pools[i] != nullptr && row > 0 && row * p->block_size <= 1 << 30, SIPA_EINVAL, "pool %d: %lld bytes a token", i,
               (long long)row);
    a.pool[i] = (char*)p->pools[i];
    a.st_l[i] = p->stride_l[i];
    a.st_h[i] = p->stride_h[i];
    a.row[i] = (int32_t)row;
    a.unit[i] = (of & 15) == 0 ? 16 : (of & 1) == 0 ? 2 : 1;
    int log = 0;  // lanes for a whole block, a workgroup at most
    while (log < 8 && (int64_t)a.unit[i] << log < row * p->block_size) ++log;
    a.log_lanes[i] = log;
    const int per = (256 >> log) * kCopyUnroll;
    most = std::max(most, (a.L * a.H + per - 1) / per);
  }
  SIPA_CHECK(most <= 65535, SIPA_EUNSUPPORTED, "%d layers of %d heads exceed the grid limit", a.L, a.H);
  for (int first = 0; first < p->num_copies; first += kCopiesPerLaunch) {
    const int n = std::min(kCopiesPerLaunch, p->num_copies - first);
    for (int i = 0; i < n; ++i) {
      const int32_t* c = p->copies + 3 * ((int64_t)first + i);
      a.src[i] = c[0], a.dst[i] = c[1], a.tokens[i] = (uint8_t)c[2];
    }
    hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)n, (unsigned)most, (unsigned)p->num_pools), dim3(256), 0,
                       (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(SIPA_EHIP, "copy of blocks failed: %s", hipGetErrorString(e));
  }
  return SIPA_OK;
}
