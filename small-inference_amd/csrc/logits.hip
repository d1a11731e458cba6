// Rules on a forward's logits before a token is taken from them: penalties for tokens already there, biases, grammar masks.
//
// The reference's engine takes the argmax of the raw logits and has no counterpart. A workgroup takes one row's `kTile`
// tokens: it counts the sequence's tokens that lie among them in LDS (integer atomics: the same counts in any order), then
// streams the logits once.
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
  const uint32_t* grammar;
  int64_t g_st;
  int32_t states;
  const int32_t* grows;
};

constexpr int kTile = 8192;                 // tokens of a workgroup: 32 KB of counts
constexpr uint32_t kSeen = 0x80000000u;     // in the prompt
constexpr uint32_t kBiased = 0x40000000u;   // in the bias list
constexpr uint32_t kCount = 0x3fffffffu;    // times made

__global__ void __launch_bounds__(256) adjust_logits_kernel(const LogitsArgs a) {
  __shared__ uint32_t cnt[kTile];
  const int r = blockIdx.y, tid = threadIdx.x;
  const int v0 = (int)blockIdx.x * kTile, n = min(kTile, a.V - v0);
  int s = r, first = r;
  if (a.qs != nullptr) {
    int lo = 0, hi = a.S;  // the last s with qs[s] <= r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.qs[mid] <= r) lo = mid; else hi = mid;
    }
    s = lo;
    first = a.qs[s];
    if (r < first || r >= a.qs[a.S]) s = -1;
  } else if (r >= a.S) {
    s = -1;
  }
  for (int i = tid; i < n; i += 256) cnt[i] = 0;
  __syncthreads();
  auto mark = [&](int64_t token, uint32_t what, bool add) {
    const int64_t i = token - v0;
    if (i < 0 || i >= n) return;
    if (add) atomicAdd(&cnt[i], what);
    else atomicOr(&cnt[i], what);
  };
  int b0 = 0, b1 = 0;
  float rho = 1.f, alpha = 0.f, beta = 0.f;
  const uint32_t* bits = nullptr;
  if (s >= 0) {
    if (a.history != nullptr) {
      const int64_t h0 = a.hstarts[s], h1 = a.hstarts[s + 1];
      const int64_t made = h0 + (a.prompt != nullptr ? max(a.prompt[s], 0) : 0);
      for (int64_t h = h0 + tid; h < h1; h += 256) mark(a.history[h], h < made ? kSeen : 1u, h >= made);
    }
    if (a.tokens != nullptr) {
      const uint64_t* m = a.masks + (int64_t)r * a.words;
      const int nodes = min(a.words * 64, (a.qs != nullptr ? a.qs[s + 1] : r + 1) - first);
      for (int i = tid; i < nodes; i += 256)
        if (m[i >> 6] >> (i & 63) & 1) mark(a.tokens[first + i], 1u, true);
    }
    if (a.bstarts != nullptr) {
      b0 = a.bstarts[s], b1 = a.bstarts[s + 1];
      for (int i = b0 + tid; i < b1; i += 256) mark(a.btok[i], kBiased, false);
    }
    if (a.rep != nullptr) rho = a.rep[s];
    if (a.freq != nullptr) alpha = a.freq[s];
    if (a.pres != nullptr) beta = a.pres[s];
    if (a.grows != nullptr) {
      const int g = a.grows[r];
      if (g >= 0 && g < a.states) bits = a.grammar + (int64_t)g * a.g_st;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const int v = v0 + i;
    float l = load_as_f32(a.logits, (int64_t)r * a.l_st + v, a.dtype);
    const uint32_t c = cnt[i];
    if (c & (kSeen | kCount)) l = l > 0.f ? l / rho : l * rho;
    if (c & kCount) l = l - alpha * (float)(c & kCount) - beta;
    if (c & kBiased) {
      float sum = 0.f;
      for (int b = b0; b < b1; ++b)
        if (a.btok[b] == v) sum += a.bval[b];
      l += sum;
    }
    if (bits != nullptr && !(bits[v >> 5] >> (v & 31) & 1)) l = -__builtin_huge_valf();
    store_from_f32(a.out, (int64_t)r * a.o_st + v, a.dtype, l);
  }
}

}  // namespace sipa

using namespace sipa;

extern "C" int32_t sipa_adjust_logits(const sipa_logits_params* p, void* stream) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_logits_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_logits_params (%d bytes)",
             (int)sizeof(sipa_logits_params));
  SIPA_CHECK(p->num_rows >= 0 && p->num_rows <= 65535 && p->vocab > 0 && p->num_seqs > 0, SIPA_EINVAL,
             "%d rows (at most 65535), vocabulary %d, %d sequences", p->num_rows, p->vocab, p->num_seqs);
  if (p->num_rows == 0) return SIPA_OK;
  SIPA_CHECK(p->dtype == SIPA_F32 || p->dtype == SIPA_BF16 || p->dtype == SIPA_F16, SIPA_EUNSUPPORTED,
             "logits of type %d", p->dtype);
  SIPA_CHECK(p->logits && p->out, SIPA_EINVAL, "NULL pointer");
  SIPA_CHECK((p->history == nullptr) == (p->history_starts == nullptr), SIPA_EINVAL, "history needs its starts");
  SIPA_CHECK((p->tokens == nullptr) == (p->masks == nullptr), SIPA_EINVAL, "a path needs tokens and masks");
  SIPA_CHECK(p->tokens == nullptr || (p->words >= 1 && p->words <= 4), SIPA_EINVAL, "%d mask words (1 .. 4)", p->words);
  SIPA_CHECK(p->bias_starts == nullptr || (p->bias_tokens && p->bias_values), SIPA_EINVAL,
             "a bias needs tokens and values");
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
  a.grammar = p->grammar;
  a.g_st = p->grammar_stride;
  a.states = p->grammar_states;
  a.grows = p->grammar_rows;
  const dim3 grid((unsigned)((p->vocab + kTile - 1) / kTile), (unsigned)p->num_rows);
  hipLaunchKernelGGL(adjust_logits_kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "logits launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}
