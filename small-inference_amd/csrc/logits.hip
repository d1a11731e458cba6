// Rules on a forward's logits before a token is taken from them: penalties for tokens already there, biases, grammar masks.
//
// The reference's engine takes the argmax of the raw logits and has no counterpart.
// The least it can do is to read and write every logit once: 512 rows of 151936 bf16 logits take 58 us as a copy and 64 here
// without any rule; histories of 5300 tokens, paths of 16 nodes, 64 biases and grammar masks bring it to 85 (3.7 TB/s). A
// workgroup of a few rows is bound by the round trips of its start (the sequence's tokens, counted in LDS).
#include <algorithm>

#include "sipa_common.h"

namespace sipa {

struct LogitsArgs {
  const void* logits;
  int64_t l_st;
  void* out;
  int64_t o_st;
  int32_t R, V, S, dtype, words;
  const int32_t* qs;
  const int32_t* history;
  const int64_t* hstarts;
  const int32_t* prompt;
  const float* rep;
  const float* freq;
  const float* pres;
  const int64_t* tokens;
  const uint64_t* masks;
  const int32_t* btok;
  const float* bval;
  const int32_t* bstarts;
  int64_t hsize;
  int32_t nbias;
  const uint32_t* grammar;
  int64_t g_st;
  int32_t states;
  const int32_t* grows;
};

constexpr uint32_t kSeen = 0x80000000u;   // in the prompt
constexpr uint32_t kPath = 0x40000000u;   // some node's token
constexpr uint32_t kCount = 0x3fffffffu;  // times among the generated tokens
constexpr int kLogitThreads = 256, kMaxNodes = 256, kTurns = 512;

template <int DT>
struct LogitsType;  // a row's element: bits, and how many make 16 bytes
template <>
struct LogitsType<SIPA_F32> {
  typedef uint32_t T;
  static constexpr int E = 4;
};
template <>
struct LogitsType<SIPA_BF16> {
  typedef uint16_t T;
  static constexpr int E = 8;
};
template <>
struct LogitsType<SIPA_F16> {
  typedef uint16_t T;
  static constexpr int E = 8;
};

template <int DT>
__device__ __forceinline__ float logit_value(uint32_t bits) {
  return DT == SIPA_F32 ? __uint_as_float(bits) : DT == SIPA_BF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32(bits);
}

// Workgroup (tile, sequence, z) takes E tokens a thread of rows z, z + Z, .. of a sequence: the sequence's tokens among them
// are counted once, in LDS, and each thread keeps its tokens' words in registers over the rows, which it streams in 16-byte
// parts (aligned to an element only: rows of an odd vocabulary start anywhere). A row's path is added to the counts before
// the row and taken out after it, by the workgroups that hold a token of it.
template <int DT>
__global__ void __launch_bounds__(kLogitThreads) adjust_logits_kernel(const LogitsArgs a) {
  typedef typename LogitsType<DT>::T T;
  constexpr int THR = kLogitThreads, E = LogitsType<DT>::E, TILE = THR * E, BITS = 8 * sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Part {
    uint32_t w[4];
  };
  __shared__ __align__(16) uint32_t cnt[TILE];
  __shared__ __align__(16) float sum[TILE];  // of the sequence's biases
  __shared__ uint32_t turn[kTurns];  // of the entries for tokens i, i + kTurns, ..: whose turn it is
  __shared__ int32_t node_token[kMaxNodes];  // within the tile, or -1
  __shared__ int32_t has_path, open_round;
  const int tid = threadIdx.x, s = blockIdx.x, v0 = (int)blockIdx.y * TILE, i0 = tid * E, n = min(TILE, a.V - v0);
  const bool behind = s >= a.S;  // (S, S + 1) rows behind the last sequence's and before the first one's: copied
  const int first = a.qs == nullptr ? s : s == a.S + 1 ? 0 : max(a.qs[s], 0);
  const int end = a.qs == nullptr ? min(s + 1, a.R) : s == a.S ? a.R : min(a.qs[s > a.S ? 0 : s + 1], a.R);
  const int r0 = first + (int)blockIdx.z;
  if (r0 >= end) return;
  const int left = n - i0;  // the thread's tokens: E of them, fewer at the vocabulary's end

  auto load = [&](int r) {
    Part x = {{0, 0, 0, 0}};
    const T* src = (const T*)a.logits + (int64_t)r * a.l_st + v0 + i0;
    if (left >= E) x = *(const Part*)src;
    else
      for (int e = 0; e < left; ++e) {
        const uint32_t bits = (uint32_t)src[e] << (BITS * e & 31);
#pragma unroll
        for (int w = 0; w < 4; ++w) x.w[w] |= BITS * e >> 5 == w ? bits : 0u;
      }
    return x;
  };
  Part x = load(r0);

  // A token's rule is l k + c, k = 1 / rho or rho by the logit's sign where it has been seen, else 1. (c = -0 where there is
  // nothing to add, so that the other logits keep their bits.)
  float inv_rho = 1.f, rho = 1.f, alpha = 0.f, beta = 0.f;
  uint32_t b0 = 0, b1 = 0;  // the sequence's biases
  uint32_t any = 0;
  float c[E];
  bool seen[E];
  auto rules = [&]() {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const uint4 w4 = *(const uint4*)(cnt + i0 + e);
      const float4 b4 = b0 < b1 ? *(const float4*)(sum + i0 + e) : float4{-0.f, -0.f, -0.f, -0.f};
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      const float bias[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float made = (float)(w[x] & kCount);
        any |= w[x] | (__float_as_uint(bias[x]) != 0x80000000u);
        seen[e + x] = (w[x] & (kSeen | kCount)) != 0;
        c[e + x] = (w[x] & kCount ? -alpha * made - beta : -0.f) + bias[x];
      }
    }
  };
#pragma unroll
  for (int e = 0; e < E; ++e) c[e] = -0.f, seen[e] = false;
  int nodes = 0;
  if (!behind) {
    const bool seq_path = a.tokens != nullptr;
    if (a.rep != nullptr) rho = a.rep[s];
    if (a.freq != nullptr) alpha = a.freq[s];
    if (a.pres != nullptr) beta = a.pres[s];
    inv_rho = 1.f / rho;
    if (a.bstarts != nullptr) b0 = max(a.bstarts[s], 0), b1 = max(min(a.bstarts[s + 1], a.nbias), 0);
#pragma unroll
    for (int i = 4 * tid; i < TILE; i += 4 * THR) {
      *(uint4*)(cnt + i) = uint4{0, 0, 0, 0};
      if (a.bstarts != nullptr) *(float4*)(sum + i) = float4{-0.f, -0.f, -0.f, -0.f};
    }
    if (a.bstarts != nullptr)
      for (int i = tid; i < kTurns; i += THR) turn[i] = 0;
    if (tid == 0) has_path = open_round = 0;
    __syncthreads();
    int entry = b0 < b1 ? a.btok[min(b0 + tid, b1 - 1)] : 0;
    if (a.history != nullptr) {
      const int64_t h0 = min(max(a.hstarts[s], (int64_t)0), a.hsize), h1 = min(a.hstarts[s + 1], a.hsize);
      const int64_t made = h0 + (a.prompt != nullptr ? max(a.prompt[s], 0) : 0);
      constexpr int U = 8, CHUNK = THR * U;  // loads in flight
      for (int64_t at = h0; at < h1; at += CHUNK) {
        const int32_t* list = a.history + at;
        const int last = (int)min(h1 - at, (int64_t)CHUNK) - 1;  // of this chunk
        const int fresh = (int)min(max(made - at, (int64_t)0), (int64_t)CHUNK);  // its first generated token
        int token[U];
#pragma unroll
        for (int u = 0; u < U; ++u) token[u] = list[min(tid + THR * u, last)];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = tid + THR * u;
          const uint32_t i = (uint32_t)token[u] - (uint32_t)v0;
          if (i >= (uint32_t)n || h > last) continue;  // (negative tokens are far past every tile)
          if (h < fresh) atomicOr(&cnt[i], kSeen);
          else atomicAdd(&cnt[i], 1u);
        }
      }
    }
    if (seq_path) {
      nodes = min(min(a.words * 64, kMaxNodes), end - first);
      if (tid < nodes) {
        const int64_t at = a.tokens[first + tid] - v0;
        const bool in = at >= 0 && at < n;
        node_token[tid] = in ? (int32_t)at : -1;
        if (in) {
          atomicOr(&cnt[at], kPath);
          has_path = 1;
        }
      }
    }
    // The biases in the list's order, THR entries at a time: of those for one token the first takes its turn (the largest
    // number), then the next, until none is left: as many rounds as some token has entries among them, mostly one (tokens
    // kTurns apart take turns too). One row and a run of 4096 neighbouring tokens: 9 us, 20000 of them 20; each biased token's
    // thread searching the list took 1950 for 4096.
    int round = 0;
    for (uint32_t at = b0; at < b1; at += THR) {
      const uint32_t i = (uint32_t)entry - (uint32_t)v0, number = THR - tid;
      bool open = i < (uint32_t)n && at + tid < b1;
      if (at + THR < b1) entry = a.btok[min(at + THR + tid, b1 - 1)];
      for (;;) {
        ++round;
        if (open) {
          open_round = round;
          atomicMax(&turn[i % kTurns], number);
        }
        __syncthreads();
        if (open_round != round) break;  // uniform: no entry was open (a thread that is ahead may have written the next round)
        if (open && turn[i % kTurns] == number) {  // (the others find this number, or the 0 after it)
          sum[i] += a.bval[at + tid];
          turn[i % kTurns] = 0;
          open = false;
        }
        __syncthreads();
      }
    }
    if (b0 >= b1) __syncthreads();  // (else the loop's last)
    rules();
  }
  const bool path = !behind && a.tokens != nullptr && has_path;  // uniform
  const int token = path && tid < nodes ? node_token[tid] : -1;
  auto on_path = [&](int r) { return token >= 0 && (a.masks[(int64_t)r * a.words + (tid >> 6)] >> (tid & 63) & 1); };
  if (path) {
    __syncthreads();  // every word has been read
    if (on_path(r0)) atomicAdd(&cnt[token], 1u);
  }
  // A row's grammar state is loaded two rows ahead of it, its bits with the row's logits one ahead.
  const bool grammar = a.grows != nullptr && !behind;
  auto state_of = [&](int r) { return grammar && r < end ? a.grows[r] : -1; };
  auto bits_of = [&](int state) {  // the thread's tokens; all ones for a free row
    const bool free = state < 0 || state >= a.states;
    const uint32_t w = free ? ~0u : a.grammar[(int64_t)state * a.g_st + (min(v0 + i0, a.V - 1) >> 5)];
    return free ? ~0u : w >> ((v0 + i0) & 31) | ~0u << E;
  };
  uint32_t allowed = bits_of(state_of(r0));
  int state = state_of(r0 + (int)gridDim.z);
  for (int r = r0; r < end; r += gridDim.z) {
    const int next = r + (int)gridDim.z;
    Part y = x;
    if (next < end) y = load(next);
    const uint32_t next_allowed = bits_of(state);
    state = state_of(next + (int)gridDim.z);
    if (path) {
      __syncthreads();  // the row's path is counted
      if (any & kPath) rules();
      __syncthreads();
      if (on_path(r)) atomicAdd(&cnt[token], ~0u);  // out again: - 1
      if (next < end && on_path(next)) atomicAdd(&cnt[token], 1u);
    }
    if (any || allowed != ~0u) {
      float l[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        l[e] = logit_value<DT>(BITS == 32 ? x.w[e] : x.w[e >> 1] >> (16 * (e & 1)) & 0xffffu);
        const float k = seen[e] ? (l[e] > 0.f ? inv_rho : rho) : 1.f;
        l[e] = fmaf(l[e], k, c[e]);
        l[e] = allowed >> e & 1 ? l[e] : -__builtin_huge_valf();
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (DT == SIPA_F32) x.w[w] = __float_as_uint(l[w]);
        else x.w[w] = DT == SIPA_BF16 ? pack_bf16x2(l[2 * w], l[2 * w + 1]) : pack_f16x2(l[2 * w], l[2 * w + 1]);
      }
    }
    T* dst = (T*)a.out + (int64_t)r * a.o_st + v0 + i0;
    if (left >= E) *(Part*)dst = x;
    else
      for (int e = 0; e < left; ++e) {
        uint32_t bits = x.w[0];
#pragma unroll
        for (int w = 1; w < 4; ++w) bits = BITS * e >> 5 == w ? x.w[w] : bits;
        dst[e] = (T)(bits >> (BITS * e & 31));
      }
    x = y;
    allowed = next_allowed;
  }
}

}  // namespace sipa

using namespace sipa;

// Tiles of 256 threads: 512 gain 1 us where every sequence has one row (32 rows 10.5 / 11.8 us) and lose more elsewhere (512
// rows 85 / 98). Rows of a sequence are shared by as many workgroups as bring the launch to 5000, three rows or more each: 32
// sequences of 16 rows 94 us with one workgroup a tile, 85 with two, 95 with three; 8 of 8 rows 17, 12 with three, 17 with
// eight.
template <int DT>
static void launch_logits(const LogitsArgs& a, hipStream_t st) {
  constexpr int TILE = kLogitThreads * LogitsType<DT>::E;
  const int64_t tiles = (a.V + TILE - 1) / TILE;
  const int64_t per = (a.R + a.S - 1) / a.S;  // rows of a sequence on average
  const int64_t z = std::max<int64_t>(1, std::min<int64_t>((per + 2) / 3, 5000 / (tiles * a.S)));
  const dim3 grid((unsigned)a.S + (a.qs != nullptr ? 2 : 0), (unsigned)tiles, (unsigned)z);  // frequent tokens first
  hipLaunchKernelGGL((adjust_logits_kernel<DT>), grid, dim3(kLogitThreads), 0, st, a);
}

extern "C" int32_t sipa_adjust_logits(const sipa_logits_params* p, void* stream) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_logits_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_logits_params (%d bytes)",
             (int)sizeof(sipa_logits_params));
  SIPA_CHECK(p->num_rows >= 0 && p->num_seqs > 0 && p->vocab > 0 && p->vocab <= 1 << 25, SIPA_EINVAL,
             "%d rows, %d sequences, vocabulary %d (up to 2^25)", p->num_rows, p->num_seqs, p->vocab);
  if (p->num_rows == 0) return SIPA_OK;
  SIPA_CHECK(p->dtype == SIPA_F32 || p->dtype == SIPA_BF16 || p->dtype == SIPA_F16, SIPA_EUNSUPPORTED,
             "logits of type %d", p->dtype);
  SIPA_CHECK(p->logits && p->out, SIPA_EINVAL, "NULL pointer");
  SIPA_CHECK((p->history == nullptr) == (p->history_starts == nullptr), SIPA_EINVAL, "history needs its starts");
  SIPA_CHECK((p->tokens == nullptr) == (p->masks == nullptr), SIPA_EINVAL, "a path needs tokens and masks");
  SIPA_CHECK(p->tokens == nullptr || (p->words >= 1 && p->words <= 4), SIPA_EINVAL, "%d mask words (1 .. 4)", p->words);
  SIPA_CHECK(p->bias_starts == nullptr || (p->bias_tokens && p->bias_values), SIPA_EINVAL,
             "a bias needs tokens and values");
  SIPA_CHECK(p->history_size >= 0 && p->num_biases >= 0, SIPA_EINVAL, "lists of negative sizes");
  SIPA_CHECK(p->grammar_rows == nullptr ||
                 (p->grammar && p->grammar_states > 0 && p->grammar_stride * 32 >= p->vocab), SIPA_EINVAL,
             "a grammar needs states of ceil(vocab / 32) words");
  LogitsArgs a;
  a.logits = p->logits;
  a.l_st = p->logits_stride;
  a.out = p->out;
  a.o_st = p->out_stride;
  a.R = p->num_rows;
  a.V = p->vocab;
  a.S = p->num_seqs;
  a.dtype = p->dtype;
  a.words = p->words;
  a.qs = p->query_starts;
  a.history = p->history;
  a.hstarts = p->history_starts;
  a.prompt = p->prompt_lens;
  a.rep = p->repetition;
  a.freq = p->frequency;
  a.pres = p->presence;
  a.tokens = p->tokens;
  a.masks = p->masks;
  a.btok = p->bias_tokens;
  a.bval = p->bias_values;
  a.bstarts = p->bias_starts;
  a.hsize = p->history_size;
  a.nbias = p->num_biases;
  a.grammar = p->grammar;
  a.g_st = p->grammar_stride;
  a.states = p->grammar_states;
  a.grows = p->grammar_rows;
  if (p->dtype == SIPA_F32) launch_logits<SIPA_F32>(a, (hipStream_t)stream);
  else if (p->dtype == SIPA_BF16) launch_logits<SIPA_BF16>(a, (hipStream_t)stream);
  else launch_logits<SIPA_F16>(a, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "logits launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}
