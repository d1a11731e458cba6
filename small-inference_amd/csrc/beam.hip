// Beams: the best continuations over the beams and the vocabulary of a request, and the copies of blocks of beams that go on
// from the same one (gfx950). The reference decodes greedily and has no counterpart.
//
// Selection, for row r (a beam) and token v:  score = cum[r] + l[r, v] - log sum_v exp(l[r, v]).  Within a row the logits
// decide the order, so that one pass over them finds a row's best tokens and its sum together:
//   beam_rows   a workgroup holds a piece of a row in registers, takes its maximum, the sum of exponentials below it, and
//               its N largest logits: those above a threshold that at least N pass (the least of the maxima of at least N
//               parts of the workgroup's lanes) are collected in LDS and put into order by counting.
//   beam_merge  a workgroup a group joins the pieces' sums in 64 bits and puts the candidates in order in the same way.
// It reads every logit once; no sum depends on the order in which workgroups or atomics run.
#include <algorithm>
#include <memory>
#include <new>

#include "decode_common.h"

namespace sipa {

constexpr int kBeamThreads = 256, kBeamMaxN = 64, kBeamMaxRows = 1024, kBeamCap = 1024, kBeamMergeCap = 512;

struct BeamArgs {
  const void* logits;
  int64_t l_st;
  const float* cum;
  const int32_t* starts;
  int32_t R, V, beams, N, ns;  // ns pieces of a row
  float* p_max;                // [R][ns]
  double* p_sum;               // [R][ns] sum of exp(l - p_max)
  float* c_val;                // [R][ns][N] a piece's largest logits in order, -inf behind them
  int32_t* c_tok;
  float* out_scores;
  int64_t* out_beams;
  int64_t* out_tokens;
};

// fp32 as an integer of the same order; of equal values the lower index is the larger key.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as 0
  return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~index;
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t x, int o) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), o) << 32 | (uint32_t)__shfl_xor((int)x, o);
}

__device__ __forceinline__ double shfl_xor_f64(double x, int o) {
  return __builtin_bit_cast(double, shfl_xor_u64(__builtin_bit_cast(uint64_t, x), o));
}

// exp(d) for d <= 0 to about an ulp: the product with log2 e is carried in two terms, since an ulp of d log2 e = 20 alone is
// 1e-6 of the result.
__device__ __forceinline__ float beam_exp(float d) {
  constexpr float kL = 1.44269502162933349609f, kLo = 1.92596299112661746887e-8f, kLn2 = 0.69314718055994530942f;
  const float y = d * kL;
  const float rest = fmaf(d, kLo, fmaf(d, kL, -y));
  const float e = fast_exp2(y);
  return y < -126.f ? 0.f : fmaf(e * kLn2, rest, e);
}

template <int DT>
struct BeamType;
template <>
struct BeamType<SIPA_F32> {
  typedef uint32_t T;
  static constexpr int E = 4;
};
template <>
struct BeamType<SIPA_BF16> {
  typedef uint16_t T;
  static constexpr int E = 8;
};
template <>
struct BeamType<SIPA_F16> {
  typedef uint16_t T;
  static constexpr int E = 8;
};

// PARTS 16-byte parts of a row a thread (aligned to an element only: rows of an odd vocabulary start anywhere).
template <int DT, int PARTS>
__global__ void __launch_bounds__(kBeamThreads) beam_rows_kernel(const BeamArgs a) {
  typedef typename BeamType<DT>::T T;
  constexpr int THR = kBeamThreads, E = BeamType<DT>::E, BITS = 8 * sizeof(T), PIECE = THR * E * PARTS;
  struct __attribute__((packed, aligned(sizeof(T)))) Part {
    uint32_t w[4];
  };
  __shared__ uint64_t found[kBeamCap];
  __shared__ float w_max[4], w_low[4];
  __shared__ double w_sum[4];
  __shared__ uint64_t w_key[4];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = blockIdx.x / a.ns, piece = blockIdx.x - r * a.ns, v0 = piece * PIECE;
  const T* row = (const T*)a.logits + (int64_t)r * a.l_st + v0;
  const int n = min(PIECE, a.V - v0);
  Part x[PARTS];
  const uint32_t kNone = DT == SIPA_F32 ? 0xff800000u : DT == SIPA_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int at = E * (tid + THR * i);
    if (at + E <= n) {
      x[i] = *(const Part*)(row + at);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) x[i].w[w] = kNone;
      for (int e = 0; e < E && at + e < n; ++e) {
        const uint32_t bits = row[at + e];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (BITS * e >> 5 == w) {
            if constexpr (BITS == 32) x[i].w[w] = bits;
            else x[i].w[w] = e & 1 ? (x[i].w[w] & 0xffffu) | bits << 16 : (x[i].w[w] & 0xffff0000u) | bits;
          }
      }
    }
  }
  auto value = [&](int i, int e) {
    if constexpr (DT == SIPA_F32) return __uint_as_float(x[i].w[e]);
    const uint32_t w = x[i].w[e >> 1];
    if constexpr (DT == SIPA_BF16) return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    return f16_bits_to_f32(e & 1 ? w >> 16 : w & 0xffffu);
  };
  auto index = [&](int i, int e) { return (uint32_t)(v0 + E * (tid + THR * i) + e); };
  float mine = kNegInf;
#pragma unroll
  for (int i = 0; i < PARTS; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) mine = fmaxf(mine, value(i, e));
  // The maxima of parts of `part` lanes each, as many parts as candidates at least, and the least of them.
  int parts = 4;
  while (parts < a.N) parts *= 2;
  const int part = THR / parts;
  float top = mine, low = mine;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    top = fmaxf(top, __shfl_xor(top, o));
    const float other = __shfl_xor(low, o);
    low = o < part ? fmaxf(low, other) : fminf(low, other);
  }
  if (lane == 0) w_max[wave] = top, w_low[wave] = low;
  if (tid == 0) count = 0;
  __syncthreads();
  top = fmaxf(fmaxf(w_max[0], w_max[1]), fmaxf(w_max[2], w_max[3]));
  low = fminf(fminf(w_low[0], w_low[1]), fminf(w_low[2], w_low[3]));
  const float off = top == kNegInf ? 0.f : top;
  double sum = 0.;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += beam_exp(value(i, e) - off);
    sum += (double)s;
  }
  if (mine >= low && mine > kNegInf) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = value(i, e);
        if (v >= low && v > kNegInf) {
          const int to = atomicAdd(&count, 1);
          if (to < kBeamCap) found[to] = beam_key(v, index(i, e));
        }
      }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += shfl_xor_f64(sum, o);
  if (lane == 0) w_sum[wave] = sum;
  __syncthreads();
  const int64_t at = (int64_t)r * a.ns + piece;
  if (tid == 0) {
    a.p_max[at] = top;
    a.p_sum[at] = (w_sum[0] + w_sum[1]) + (w_sum[2] + w_sum[3]);
  }
  int got = count;
  float* c_val = a.c_val + at * a.N;
  int32_t* c_tok = a.c_tok + at * a.N;
  if (got <= kBeamCap) {
    for (int i = tid; i < got; i += THR) {
      const uint64_t key = found[i];
      int rank = 0;
      for (int j = 0; j < got; ++j) rank += found[j] > key;
      if (rank < a.N) c_val[rank] = key_value(key), c_tok[rank] = (int32_t)~(uint32_t)key;
    }
  } else {
    // Most of the piece ties or rises: the largest key under the last one, N times. Only the thread that had it looks for
    // its next.
    auto best_below = [&](uint64_t limit) {
      uint64_t best = 0;
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float v = value(i, e);
          const uint64_t key = v > kNegInf ? beam_key(v, index(i, e)) : 0;
          best = key < limit && key > best ? key : best;
        }
      return best;
    };
    uint64_t own = best_below(~0ull);
    got = 0;
    for (int k = 0; k < a.N; ++k) {
      uint64_t best = own;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t other = shfl_xor_u64(best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) w_key[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w) best = w_key[w] > best ? w_key[w] : best;
      __syncthreads();
      if (best == 0) break;  // uniform
      if (own == best) {
        c_val[k] = key_value(best), c_tok[k] = (int32_t)~(uint32_t)best;
        own = best_below(best);
      }
      ++got;
    }
  }
  for (int i = got + tid; i < a.N; i += THR) c_val[i] = kNegInf, c_tok[i] = -1;
}

// A candidate of a group: its score's bits in order, its row within the group, its logit and token (beam_key). Equal scores go
// by row, then as the row orders its tokens: logits so small that they leave no trace in the score still do that.
struct BeamCandidate {
  uint64_t score, key;
  uint32_t row;
  __device__ __forceinline__ bool over(const BeamCandidate& o) const {
    return score != o.score ? score > o.score : row != o.row ? row < o.row : key > o.key;
  }
};

__device__ __forceinline__ uint64_t f64_order(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.);
  return b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ double order_f64(uint64_t b) {
  return __builtin_bit_cast(double, b >> 63 ? b & ~(1ull << 63) : ~b);
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamArgs a) {
  constexpr int THR = kBeamThreads;
  __shared__ double offset[kBeamMaxRows];  // cum - log sum exp, NaN for a row without candidates
  __shared__ BeamCandidate found[kBeamMergeCap];
  __shared__ uint64_t w_low[4];
  __shared__ BeamCandidate w_best[4];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = blockIdx.x;
  const int r0 = a.starts == nullptr ? g * a.beams : min(max(a.starts[g], 0), a.R);
  const int r1 = a.starts == nullptr ? r0 + a.beams : min(max(a.starts[g + 1], r0), a.R);
  const int rows = min(r1 - r0, kBeamMaxRows);
  for (int b = wave; b < rows; b += 4) {  // a wave a row
    const int64_t first = (int64_t)(r0 + b) * a.ns;
    float top = kNegInf;
    for (int i = lane; i < a.ns; i += 64) top = fmaxf(top, a.p_max[first + i]);
    top = wave_max(top);
    double sum = 0.;
    for (int i = lane; i < a.ns; i += 64) {
      const float m = a.p_max[first + i];
      const double s = a.p_sum[first + i];
      sum += m == kNegInf ? s : s * exp((double)m - (double)top);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += shfl_xor_f64(sum, o);
    const double lse = (double)top + log(sum), cum = (double)a.cum[r0 + b];
    const double off = cum - lse;
    if (lane == 0) offset[b] = fabs(off) < __builtin_huge_val() ? off : __builtin_nan("");
  }
  if (tid == 0) count = 0;
  __syncthreads();
  const int per = a.ns * a.N, total = rows * per;  // (host-checked)
  const int64_t first = (int64_t)r0 * per;
  auto candidate = [&](int i) {
    const int b = i / per;
    const float v = a.c_val[first + i];
    const double s = offset[b] + (double)v;
    BeamCandidate c;
    c.score = s > -__builtin_huge_val() ? f64_order(s) : 0;  // 0: none (-inf, NaN)
    c.key = beam_key(v, (uint32_t)a.c_tok[first + i]);
    c.row = (uint32_t)b;
    return c;
  };
  // The threshold, as in beam_rows.
  uint64_t mine = 0;
  for (int i = tid; i < total; i += THR) {
    const uint64_t s = candidate(i).score;
    mine = s > mine ? s : mine;
  }
  int parts = 4;
  while (parts < a.N) parts *= 2;
  const int part = THR / parts;
  uint64_t low = mine;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint64_t other = shfl_xor_u64(low, o);
    low = (o < part) == (other > low) ? other : low;
  }
  if (lane == 0) w_low[wave] = low;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) low = w_low[w] < low ? w_low[w] : low;
  if (mine >= low && mine > 0)
    for (int i = tid; i < total; i += THR) {
      const BeamCandidate c = candidate(i);
      if (c.score >= low && c.score > 0) {
        const int to = atomicAdd(&count, 1);
        if (to < kBeamMergeCap) found[to] = c;
      }
    }
  __syncthreads();
  int got = count;
  const int64_t out = (int64_t)g * a.N;
  auto store = [&](int k, const BeamCandidate& c) {
    a.out_scores[out + k] = (float)order_f64(c.score);
    a.out_beams[out + k] = (int64_t)c.row;
    a.out_tokens[out + k] = (int64_t)(uint32_t)~(uint32_t)c.key;
  };
  if (got <= kBeamMergeCap) {
    for (int i = tid; i < got; i += THR) {
      const BeamCandidate c = found[i];
      int rank = 0;
      for (int j = 0; j < got; ++j) rank += found[j].over(c);
      if (rank < a.N) store(rank, c);
    }
  } else {
    const BeamCandidate kNone = {0, 0, ~0u};
    auto best_below = [&](const BeamCandidate& limit, bool all) {
      BeamCandidate best = kNone;
      for (int i = tid; i < total; i += THR) {
        const BeamCandidate c = candidate(i);
        if (c.score > 0 && (all || limit.over(c)) && c.over(best)) best = c;
      }
      return best;
    };
    BeamCandidate own = best_below(kNone, true);
    got = 0;
    for (int k = 0; k < a.N; ++k) {
      BeamCandidate best = own;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const BeamCandidate other = {shfl_xor_u64(best.score, o), shfl_xor_u64(best.key, o), (uint32_t)__shfl_xor((int)best.row, o)};
        if (other.over(best)) best = other;
      }
      if (lane == 0) w_best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (w_best[w].over(best)) best = w_best[w];
      __syncthreads();
      if (best.score == 0) break;  // uniform
      if (own.score == best.score && own.key == best.key && own.row == best.row) {
        store(k, best);
        own = best_below(best, false);
      }
      ++got;
    }
  }
  for (int i = got + tid; i < a.N; i += THR) {
    a.out_scores[out + i] = kNegInf;
    a.out_beams[out + i] = a.out_tokens[out + i] = -1;
  }
}

// ---- copies of blocks --------------------------------------------------------------------------------------------------

constexpr int kCopiesPerLaunch = 256, kCopyPools = 4, kCopyUnroll = 4;

struct CopyArgs {
  char* pool[kCopyPools];
  int64_t st_l[kCopyPools], st_h[kCopyPools];
  int32_t row[kCopyPools];         // bytes of a token
  int32_t unit[kCopyPools];        // bytes moved at a time
  int32_t log_lanes[kCopyPools];   // lanes of a (layer, head)
  int32_t L, H, B;
  int32_t src[kCopiesPerLaunch], dst[kCopiesPerLaunch];
  uint16_t tokens[kCopiesPerLaunch];
};

// Workgroup (copy, y, pool): (layer, head) segments of one block, 1 << log_lanes lanes side by side on each.
template <typename U>
__device__ __forceinline__ void copy_segments(const CopyArgs& a, int pool, int c) {
  const int lanes = 1 << a.log_lanes[pool], per = (256 >> a.log_lanes[pool]), lane = threadIdx.x & (lanes - 1);
  const int units = (int)((int64_t)a.tokens[c] * a.row[pool] / (int)sizeof(U)), all = a.L * a.H;
  const int64_t block = (int64_t)a.B * a.row[pool];
  const int first = blockIdx.y * per * kCopyUnroll + (threadIdx.x >> a.log_lanes[pool]);
  if (first >= all) return;
  for (int u = lane; u < units; u += lanes) {
    U x[kCopyUnroll];
    char* at[kCopyUnroll];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i) {
      const int seg = min(first + per * i, all - 1), l = seg / a.H;
      at[i] = a.pool[pool] + l * a.st_l[pool] + (seg - l * a.H) * a.st_h[pool];
      x[i] = *((const U*)(at[i] + a.src[c] * block) + u);
    }
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
      if (first + per * i < all) *((U*)(at[i] + a.dst[c] * block) + u) = x[i];
  }
}

__global__ void __launch_bounds__(256) copy_blocks_kernel(const CopyArgs a) {
  const int pool = blockIdx.z, c = blockIdx.x;
  if (a.unit[pool] == 16) copy_segments<uint4>(a, pool, c);
  else if (a.unit[pool] == 2) copy_segments<uint16_t>(a, pool, c);
  else copy_segments<uint8_t>(a, pool, c);
}

}  // namespace sipa

using namespace sipa;

// Pieces of a row: parts of a thread, by type.
static int beam_parts(const sipa_beam_params* p) {
  const int e = p->dtype == SIPA_F32 ? 4 : 8;
  for (int parts = 8; parts > 1; parts /= 2)
    if ((int64_t)p->num_rows * ((p->vocab + kBeamThreads * e * parts - 1) / (kBeamThreads * e * parts)) >= 512) return parts;
  return 1;
}

struct BeamLayout {
  int parts, ns;
  int64_t sum, val, tok, total;
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
  const int piece = kBeamThreads * (p->dtype == SIPA_F32 ? 4 : 8) * l->parts;
  l->ns = (p->vocab + piece - 1) / piece;
  const int64_t pieces = (int64_t)p->num_rows * l->ns;
  SIPA_CHECK(pieces <= 0x7fffffff && (int64_t)std::min(p->num_rows, kBeamMaxRows) * l->ns * p->num_candidates <= 0x7fffffff,
             SIPA_EUNSUPPORTED, "%d rows of %d pieces exceed the grid limit", p->num_rows, l->ns);
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  l->sum = up(pieces * 4);
  l->val = l->sum + up(pieces * 8);
  l->tok = l->val + up(pieces * p->num_candidates * 4);
  l->total = l->tok + up(pieces * p->num_candidates * 4);
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
  else if (parts == 2) hipLaunchKernelGGL((beam_rows_kernel<DT, 2>), dim3(grid), dim3(kBeamThreads), 0, st, a);
  else hipLaunchKernelGGL((beam_rows_kernel<DT, 1>), dim3(grid), dim3(kBeamThreads), 0, st, a);
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
  char* ws = (char*)p->workspace;
  a.p_max = (float*)ws;
  a.p_sum = (double*)(ws + l.sum);
  a.c_val = (float*)(ws + l.val);
  a.c_tok = (int32_t*)(ws + l.tok);
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
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)p->num_groups), dim3(kBeamThreads), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "beam selection launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}

extern "C" int32_t sipa_check_copies(const int32_t* copies, int32_t num_copies, int32_t num_blocks, int32_t block_size) {
  SIPA_CHECK(num_copies >= 0 && num_blocks >= 0 && block_size > 0, SIPA_EINVAL, "%d copies, %d blocks of %d tokens", num_copies,
             num_blocks, block_size);
  if (num_copies == 0) return SIPA_OK;
  SIPA_CHECK(copies != nullptr, SIPA_EINVAL, "NULL pointer");
  // every block with 1 where it is a destination, in order: equal neighbours that are not both sources collide
  constexpr int kHere = 256;
  uint64_t here[2 * kHere];
  std::unique_ptr<uint64_t[]> more;
  uint64_t* of = here;
  if (num_copies > kHere) {
    more.reset(new (std::nothrow) uint64_t[2 * (size_t)num_copies]);
    SIPA_CHECK(more != nullptr, SIPA_EINVAL, "no memory for %d copies", num_copies);
    of = more.get();
  }
  for (int i = 0; i < num_copies; ++i) {
    const int32_t* c = copies + 3 * (int64_t)i;
    SIPA_CHECK(c[0] >= 0 && c[0] < num_blocks && c[1] >= 0 && c[1] < num_blocks && c[2] >= 0 && c[2] <= block_size,
               SIPA_EINVAL, "copy %d: %d tokens of block %d to block %d (%d blocks of %d tokens)", i, c[2], c[0], c[1],
               num_blocks, block_size);
    of[2 * (int64_t)i] = 2 * (uint64_t)c[0], of[2 * (int64_t)i + 1] = 2 * (uint64_t)c[1] + 1;
  }
  std::sort(of, of + 2 * (int64_t)num_copies);
  for (int64_t i = 1; i < 2 * (int64_t)num_copies; ++i)
    SIPA_CHECK(of[i] >> 1 != of[i - 1] >> 1 || of[i] % 2 == 0, SIPA_EINVAL,
               "block %lld is the destination of two copies, or of one and the source of another", (long long)(of[i] >> 1));
  return SIPA_OK;
}

extern "C" int32_t sipa_copy_blocks(const sipa_copy_params* p, void* stream) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_copy_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_copy_params (%d bytes)", (int)sizeof(sipa_copy_params));
  SIPA_CHECK(p->num_layers >= 0 && p->num_kv_heads >= 0 && p->num_blocks >= 0 && p->block_size > 0 && p->block_size <= 65535 &&
                 p->num_copies >= 0 && p->num_pools >= 1 && p->num_pools <= kCopyPools &&
                 (int64_t)p->num_layers * p->num_kv_heads <= 1 << 24, SIPA_EINVAL,
             "%d layers of %d heads, %d blocks of %d tokens, %d pools, %d copies", p->num_layers, p->num_kv_heads, p->num_blocks,
             p->block_size, p->num_pools, p->num_copies);
  if (p->num_copies == 0 || p->num_layers == 0 || p->num_kv_heads == 0) return SIPA_OK;
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
    int log = 0;  // lanes for a whole block, a wave at most
    while (log < 6 && (int64_t)a.unit[i] << log < row * p->block_size) ++log;
    a.log_lanes[i] = log;
    const int per = (256 >> log) * kCopyUnroll;
    most = std::max(most, (a.L * a.H + per - 1) / per);
  }
  SIPA_CHECK(most <= 65535, SIPA_EUNSUPPORTED, "%d layers of %d heads exceed the grid limit", a.L, a.H);
  for (int first = 0; first < p->num_copies; first += kCopiesPerLaunch) {
    const int n = std::min(kCopiesPerLaunch, p->num_copies - first);
    for (int i = 0; i < n; ++i) {
      const int32_t* c = p->copies + 3 * ((int64_t)first + i);
      a.src[i] = c[0], a.dst[i] = c[1], a.tokens[i] = (uint16_t)c[2];
    }
    hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)n, (unsigned)most, (unsigned)p->num_pools), dim3(256), 0,
                       (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(SIPA_EHIP, "copy of blocks failed: %s", hipGetErrorString(e));
  }
  return SIPA_OK;
}
