// Attention of drafted trees over the paged cache on the matrix cores (gfx950).
//
// A sequence's n nodes, each with G query heads for a KV head, make n G rows that read the same keys; row m is node m / G,
// head m % G, so that small trees fill whole 16-row tiles whatever the group size. A row sees the sequence's cached tokens
// and the nodes in its mask. The reference has no counterpart: it decodes one token per step.
//
// Work unit: (sequence, KV head, kRows rows); its keys are cut into splits of `chunk`, one workgroup each. The workgroup
// brings 32 keys at a time into LDS, each of its waves takes 16 rows:
//   S^T[16 keys x 16 rows] = K[16 x 32 d] . Q^T[32 d x 16 rows]   v_mfma_f32_16x16x32_bf16
//   hidden keys -> -inf; online softmax per row in the exp2 domain
//   O^T[16 d x 16 rows] += V^T . P^T
// INT8 pools: the codes go to LDS as bf16, exactly; the scores are multiplied by K's scales and the probabilities by V's in
// fp32. Splits write (m, l, O) and the last of a unit's to arrive merges them.
// P is rounded to bf16 for the second product, as the model's own attention rounds its probabilities (2^-9 of each, which
// averages out over the keys): V has no more bits, and a second term would double that product.
#include <algorithm>

#include "decode_common.h"

namespace sipa {

constexpr int kTreeRows = 64;         // rows of a workgroup: 4 waves of 16
constexpr int kTreeMaxSplits = 128;
constexpr int kTreeMaxChunk = 32768;
constexpr int kTreeMaxGroup = 64;
constexpr int kTreeMaxNodes = 256;

struct TreeArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const void* k;
  const void* v;
  int64_t kv_sh, kv_sn;
  const int32_t* bt;
  int64_t bt_ss;
  int32_t bt_w;
  const int32_t* ctx;
  const int32_t* qs;
  const uint64_t* masks;
  uint16_t* out;
  int64_t o_st, o_sh;
  const void* ks;
  const void* vs;
  bool ks_f32, vs_f32;
  int64_t ks_sh, ks_sn, vs_sh, vs_sn;
  int32_t S, T, Hkv, G, words, nb, max_ctx, max_nodes;
  int32_t log_b;           // blocks of 1 << log_b tokens
  int32_t groups;          // row groups of the longest sequence
  int32_t units, nsplit, chunk;
  float scale_log2;
  int* counters;           // [units]
  float* pm;               // [units][nsplit][kTreeRows]
  float* pl;
  float* part;             // [units][nsplit][kTreeRows][D]
};

__device__ __forceinline__ float tree_scale(const void* base, bool f32, int64_t i) {
  return f32 ? ((const float*)base)[i] : f16_bits_to_f32(((const uint16_t*)base)[i]);
}

template <int D, int MODE>
__global__ void __launch_bounds__(256) tree_attention_kernel(const TreeArgs a) {
  constexpr int KT = 32, P = D + 16, KS = D / 32, DT = D / 16;
  constexpr int CH = MODE == 0 ? 8 : 16, CPK = D / CH, LPT = (KT * CPK + 255) / 256;  // 16-byte parts of a tile
  __shared__ __align__(16) uint16_t sk[KT * P];
  __shared__ __align__(16) uint16_t sv[KT * P];
  __shared__ float sks[KT], svs[KT];
  __shared__ int last_flag;

  const int u = (int)blockIdx.x % a.units, sp = (int)blockIdx.x / a.units;
  const int rg = u % a.groups, s = u / a.groups % a.S, h = u / a.groups / a.S;
  const int row0 = a.qs[s], n = min(min(a.qs[s + 1] - row0, a.max_nodes), a.T - row0);
  const int G = a.G, M = n * G, m0 = rg * kTreeRows;
  if (n <= 0 || row0 < 0 || m0 >= M) return;
  const int ctx = min(a.ctx[s], a.max_ctx), start = ctx - (a.qs[s + 1] - row0);
  const int nvalid = max(1, (ctx + a.chunk - 1) / a.chunk);
  if (sp >= nvalid) return;
  const int k_lo = sp * a.chunk, k_hi = min(k_lo + a.chunk, ctx);

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q4 = lane >> 4;
  const int m = m0 + 16 * wave + r;
  const bool valid = m < M;
  const int node = (valid ? m : M - 1) / G, g = (valid ? m : M - 1) - node * G;
  bf16x8 qop[KS];
#pragma unroll
  for (int j = 0; j < KS; ++j)
    qop[j] = __builtin_bit_cast(bf16x8, *(const u32x4*)(a.q + (int64_t)(row0 + node) * a.q_st +
                                                        (int64_t)(h * G + g) * a.q_sh + 32 * j + 8 * q4));
  const uint64_t* mask = a.masks + (int64_t)(row0 + node) * a.words;
  float m_run = kNegInf, l_run = 0.f;
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int tr_off = tr16_offset(r, q4, P);

  for (int t0 = k_lo; t0 < k_hi; t0 += KT) {
    __syncthreads();  // the tile before this one is done with
#pragma unroll
    for (int i = 0; i < LPT; ++i) {
      const int c = tid + 256 * i;
      if (c >= KT * CPK) break;
      const int key = c / CPK, d0 = CH * (c % CPK), pos = min(t0 + key, k_hi - 1);
      const int64_t blk = min(max(a.bt[(int64_t)s * a.bt_ss + min(pos >> a.log_b, a.bt_w - 1)], 0), a.nb - 1);
      const int off = pos & ((1 << a.log_b) - 1);
      const int64_t e = (int64_t)h * a.kv_sh + blk * a.kv_sn + (int64_t)off * D + d0;
      if constexpr (MODE == 0) {
        *(u32x4*)(sk + key * P + d0) = *(const u32x4*)((const uint16_t*)a.k + e);
        *(u32x4*)(sv + key * P + d0) = *(const u32x4*)((const uint16_t*)a.v + e);
      } else {
        const u32x4 k = *(const u32x4*)((const int8_t*)a.k + e), v = *(const u32x4*)((const int8_t*)a.v + e);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int b = 0; b < 4; b += 2) {
            *(uint32_t*)(sk + key * P + d0 + 4 * w + b) =
                pack_bf16x2((float)(int8_t)(k[w] >> (8 * b)), (float)(int8_t)(k[w] >> (8 * b + 8)));
            *(uint32_t*)(sv + key * P + d0 + 4 * w + b) =
                pack_bf16x2((float)(int8_t)(v[w] >> (8 * b)), (float)(int8_t)(v[w] >> (8 * b + 8)));
          }
        if (d0 == 0) {
          sks[key] = tree_scale(a.ks, a.ks_f32, (int64_t)h * a.ks_sh + blk * a.ks_sn + off);
          svs[key] = tree_scale(a.vs, a.vs_f32, (int64_t)h * a.vs_sh + blk * a.vs_sn + off);
        }
      }
    }
    __syncthreads();
    float sc[8];  // keys 16 (i / 4) + 4 q4 + i % 4 of the tile
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j)
        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)(sk + (16 * mt + r) * P + 32 * j + 8 * q4), qop[j],
                                                    x, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[4 * mt + i] = MODE == 0 ? x[i] : x[i] * sks[16 * mt + 4 * q4 + i];
    }
    const bool masked = t0 + KT > min(start, k_hi);  // some key of the tile is a node, or past the split's end
    if (masked) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = t0 + 16 * (i >> 2) + 4 * q4 + (i & 3), rel = key - start;
        bool sees = key < k_hi;
        if (rel >= 0) sees = sees && rel < 64 * a.words && (mask[rel >> 6] >> (rel & 63) & 1);
        if (!sees) sc[i] = kNegInf;
      }
    }
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = vmax(mx, sc[i]);
    mx = max_over_rows_swap(mx) * a.scale_log2;
    const float m_new = vmax(m_run, mx), base = m_new == kNegInf ? 0.f : m_new;
    const float alpha = fast_exp2(m_run - base);  // 0 while the row has seen no key
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
    bf16x8 pop;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = fast_exp2(fmaf(sc[i], a.scale_log2, -base));
      l_run += p[i];
      if constexpr (MODE == 1) {
        const float scaled = p[i] * svs[16 * (i >> 2) + 4 * q4 + (i & 3)];
        p[i] = masked && p[i] == 0.f ? 0.f : scaled;  // a hidden key's scale may be anything
      }
      pop[i] = (__bf16)p[i];
    }
    // Infinities and NaN among the nodes' V: rows that do not see them must not take 0 * V into their sums.
    bool plain = true;
    if (MODE == 0 && masked) {
      bool bad = false;
      for (int c = lane; c < KT * D / 2; c += 64) {
        const uint32_t w = *(const uint32_t*)(sv + (2 * c / D) * P + 2 * c % D);
        bad = bad || (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
      }
      plain = __builtin_amdgcn_ballot_w64(bad) == 0;
    }
    if (plain) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(read_v_operand<bf16x8>(sv, tr_off, P, 16 * dt), pop, acc[dt], 0,
                                                          0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        for (int from = 0; from < 4; ++from) {  // lane group `from` holds the probability of this key
          const float pk = __shfl((float)pop[i], 16 * from + r);
          const uint16_t* v = sv + (16 * (i >> 2) + 4 * from + (i & 3)) * P;
          if (pk != 0.f)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[dt][e] += pk * bf16_bits_to_f32(v[16 * dt + 4 * q4 + e]);
        }
    }
  }
  const float l = sum_over_rows_swap(l_run);
  if (nvalid == 1) {
    if (!valid) return;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros
    uint16_t* o = a.out + (int64_t)(row0 + node) * a.o_st + (int64_t)(h * G + g) * a.o_sh + 4 * q4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint32_t* w = (uint32_t*)(o + 16 * dt);
      w[0] = pack_bf16x2(acc[dt][0] * inv, acc[dt][1] * inv);
      w[1] = pack_bf16x2(acc[dt][2] * inv, acc[dt][3] * inv);
    }
    return;
  }
  const int64_t base = ((int64_t)u * a.nsplit + sp) * kTreeRows;
  const int slot = 16 * wave + r;
  const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(
      a.part + (int64_t)u * a.nsplit * kTreeRows * D, (short)0, a.nsplit * kTreeRows * D * 4, 0x00020000);
  if (valid) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[dt]), rows,
                                             ((sp * kTreeRows + slot) * D + 16 * dt + 4 * q4) * 4, 0, kAuxSc1);
    if (q4 == 0) {
      store_coherent(a.pm + base + slot, m_run);
      store_coherent(a.pl + base + slot, l);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    last_flag = __hip_atomic_fetch_add(a.counters + u, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nvalid - 1;
  __syncthreads();
  if (!last_flag) return;
  const int64_t first = (int64_t)u * a.nsplit * kTreeRows;
  for (int i = tid; i < kTreeRows * (D / 4); i += 256) {
    const int row = i / (D / 4), c = i % (D / 4);
    if (m0 + row >= M) break;
    float top = kNegInf, den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < nvalid; ++j) {
      const float mj = load_coherent(a.pm + first + j * kTreeRows + row), lj = load_coherent(a.pl + first + j * kTreeRows + row);
      const f32x4 oj = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, ((j * kTreeRows + row) * D + 4 * c) * 4, 0, kAuxSc1));
      if (mj == kNegInf && lj == 0.f) continue;  // the row sees no key of this split
      const float up = vmax(top, mj), f = fast_exp2(top - up), w = fast_exp2(mj - up);
      den = den * f + lj * w;
      num = num * f + oj * w;
      top = up;
    }
    const float inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);
    const int nd = (m0 + row) / G, hd = (m0 + row) - nd * G;
    uint32_t* w = (uint32_t*)(a.out + (int64_t)(row0 + nd) * a.o_st + (int64_t)(h * G + hd) * a.o_sh + 4 * c);
    w[0] = pack_bf16x2(num[0] * inv, num[1] * inv);
    w[1] = pack_bf16x2(num[2] * inv, num[3] * inv);
  }
  if (tid == 0) __hip_atomic_store(a.counters + u, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace sipa

using namespace sipa;

struct TreeLayout {
  int groups, units, nsplit, chunk;
  int64_t pm, pl, part, total;  // byte offsets into the workspace; counters first
};

static int tree_check(const sipa_tree_params* p) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_tree_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_tree_params (%d bytes)", (int)sizeof(sipa_tree_params));
  SIPA_CHECK(p->num_seqs >= 0 && p->num_tokens >= 0 && p->num_kv_heads > 0 && p->num_q_heads > 0 &&
                 p->num_q_heads % p->num_kv_heads == 0, SIPA_EINVAL, "bad sequence, token or head counts");
  SIPA_CHECK(p->num_q_heads / p->num_kv_heads <= kTreeMaxGroup, SIPA_EUNSUPPORTED, "GQA group %d > %d",
             p->num_q_heads / p->num_kv_heads, kTreeMaxGroup);
  SIPA_CHECK(p->head_dim == 64 || p->head_dim == 128, SIPA_EUNSUPPORTED, "head_dim %d not in {64, 128}", p->head_dim);
  SIPA_CHECK(p->block_size == 16 || p->block_size == 32 || p->block_size == 64, SIPA_EUNSUPPORTED,
             "block_size %d not in {16, 32, 64}", p->block_size);
  SIPA_CHECK(p->max_context > 0 && p->max_context <= kTreeMaxSplits * kTreeMaxChunk, SIPA_EUNSUPPORTED,
             "max_context %d outside [1, %d]", p->max_context, kTreeMaxSplits * kTreeMaxChunk);
  SIPA_CHECK(p->max_nodes > 0 && p->max_nodes <= kTreeMaxNodes, SIPA_EUNSUPPORTED, "trees of %d nodes (1 .. %d)",
             p->max_nodes, kTreeMaxNodes);
  SIPA_CHECK(p->words >= 1 && p->words <= 4 && p->max_nodes <= 64 * p->words, SIPA_EINVAL,
             "masks of %d words for trees of %d nodes", p->words, p->max_nodes);
  SIPA_CHECK(p->kv_mode == SIPA_KV_PLAIN || p->kv_mode == SIPA_KV_INT8_TOKEN, SIPA_EUNSUPPORTED, "kv_mode %d",
             p->kv_mode);
  return SIPA_OK;
}

// About two workgroups per CU, splits of at least 256 keys.
static int tree_layout(const sipa_tree_params* p, TreeLayout* l) {
  const int G = p->num_q_heads / p->num_kv_heads;
  l->groups = (p->max_nodes * G + kTreeRows - 1) / kTreeRows;
  const int64_t units = (int64_t)p->num_seqs * p->num_kv_heads * l->groups;
  SIPA_CHECK(units <= 0x7fffffff / kTreeMaxSplits, SIPA_EINVAL, "%lld units exceed the grid limit", (long long)units);
  l->units = (int)units;
  int64_t splits = p->num_splits;
  if (splits <= 0) {
    const int cus = sipa_device_cu_count(-1);
    if (cus < 0) return cus;
    splits = std::min<int64_t>((2 * cus + units - 1) / std::max<int64_t>(units, 1), (p->max_context + 255) / 256);
  }
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, kTreeMaxSplits));
  const int chunk = (int)((p->max_context + splits - 1) / splits);
  l->chunk = std::min((chunk + 63) / 64 * 64, kTreeMaxChunk);
  l->nsplit = (p->max_context + l->chunk - 1) / l->chunk;
  l->pm = l->pl = l->part = l->total = 0;
  if (l->nsplit > 1) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t rows = units * l->nsplit * kTreeRows;
    SIPA_CHECK((int64_t)l->nsplit * kTreeRows * p->head_dim * 4 <= 0x7fffffff, SIPA_EINVAL, "split state too large");
    l->pm = up(units * 4);
    l->pl = l->pm + up(rows * 4);
    l->part = l->pl + up(rows * 4);
    l->total = l->part + up(rows * p->head_dim * 4);
  }
  return SIPA_OK;
}

extern "C" int64_t sipa_tree_workspace_bytes(const sipa_tree_params* p, int64_t* counter_bytes) {
  if (counter_bytes != nullptr) *counter_bytes = 0;
  int rc = tree_check(p);
  if (rc != SIPA_OK) return rc;
  TreeLayout l;
  rc = tree_layout(p, &l);
  if (rc != SIPA_OK) return rc;
  if (counter_bytes != nullptr) *counter_bytes = l.pm;
  return l.total;
}

extern "C" uint64_t sipa_capture_id(void* stream) {
  if (stream == nullptr) return 0;  // the default stream is never captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusNone ? 0 : (uint64_t)id;
}

extern "C" int32_t sipa_tree_attention(const sipa_tree_params* p, void* stream) {
  int rc = tree_check(p);
  if (rc != SIPA_OK) return rc;
  if (p->num_seqs == 0 || p->num_tokens == 0) return SIPA_OK;
  SIPA_CHECK(p->scale > 0.f && p->scale < __builtin_inff(), SIPA_EINVAL,
             "scale %g must be positive and finite (the kernel takes maxima of the unscaled scores)", (double)p->scale);
  SIPA_CHECK(p->bt_width > 0 && (int64_t)p->bt_width * p->block_size >= p->max_context, SIPA_EINVAL,
             "block_tables rows of %d entries cannot cover max_context %d", p->bt_width, p->max_context);
  SIPA_CHECK(p->q && p->k_cache && p->v_cache && p->block_tables && p->context_lens && p->query_starts && p->masks &&
                 p->out && p->num_blocks > 0, SIPA_EINVAL, "NULL pointer or empty pool");
  SIPA_CHECK(((uintptr_t)p->q & 15) == 0 && p->q_stride_t % 8 == 0 && p->q_stride_h % 8 == 0, SIPA_EINVAL,
             "q rows must be 16-byte aligned");
  SIPA_CHECK(((uintptr_t)p->out & 15) == 0 && p->out_stride_t % 8 == 0 && p->out_stride_h % 8 == 0, SIPA_EINVAL,
             "out rows must be 16-byte aligned");
  const bool int8 = p->kv_mode == SIPA_KV_INT8_TOKEN;
  const int per16 = int8 ? 16 : 8;
  SIPA_CHECK((((uintptr_t)p->k_cache | (uintptr_t)p->v_cache) & 15) == 0 && p->kv_stride_h % per16 == 0 &&
                 p->kv_stride_n % per16 == 0, SIPA_EINVAL, "K/V pools must be 16-byte aligned");
  if (int8) {
    SIPA_CHECK(p->k_scale && p->v_scale, SIPA_EINVAL, "INT8 pools need k_scale and v_scale");
    SIPA_CHECK((p->k_scale_dtype == SIPA_F16 || p->k_scale_dtype == SIPA_F32) &&
                   (p->v_scale_dtype == SIPA_F16 || p->v_scale_dtype == SIPA_F32),
               SIPA_EUNSUPPORTED, "scales must be fp16 or fp32");
    SIPA_CHECK(((uintptr_t)p->k_scale % (p->k_scale_dtype == SIPA_F32 ? 4 : 2)) == 0 &&
                   ((uintptr_t)p->v_scale % (p->v_scale_dtype == SIPA_F32 ? 4 : 2)) == 0, SIPA_EINVAL,
               "scales must be aligned to their element size");
  }
  TreeLayout l;
  rc = tree_layout(p, &l);
  if (rc != SIPA_OK) return rc;
  SIPA_CHECK(l.total == 0 || (p->workspace != nullptr && ((uintptr_t)p->workspace & 255) == 0 &&
                              p->workspace_bytes >= l.total),
             SIPA_EWORKSPACE, "%d key splits need a 256-byte aligned workspace of %lld bytes (have %lld)", l.nsplit,
             (long long)l.total, (long long)p->workspace_bytes);
  TreeArgs a;
  a.q = (const uint16_t*)p->q;
  a.q_st = p->q_stride_t;
  a.q_sh = p->q_stride_h;
  a.k = p->k_cache;
  a.v = p->v_cache;
  a.kv_sh = p->kv_stride_h;
  a.kv_sn = p->kv_stride_n;
  a.bt = p->block_tables;
  a.bt_ss = p->bt_stride_s;
  a.bt_w = p->bt_width;
  a.ctx = p->context_lens;
  a.qs = p->query_starts;
  a.masks = p->masks;
  a.out = (uint16_t*)p->out;
  a.o_st = p->out_stride_t;
  a.o_sh = p->out_stride_h;
  a.ks = p->k_scale;
  a.vs = p->v_scale;
  a.ks_f32 = p->k_scale_dtype == SIPA_F32;
  a.vs_f32 = p->v_scale_dtype == SIPA_F32;
  a.ks_sh = p->ks_stride_h;
  a.ks_sn = p->ks_stride_n;
  a.vs_sh = p->vs_stride_h;
  a.vs_sn = p->vs_stride_n;
  a.S = p->num_seqs;
  a.T = p->num_tokens;
  a.Hkv = p->num_kv_heads;
  a.G = p->num_q_heads / p->num_kv_heads;
  a.words = p->words;
  a.nb = p->num_blocks;
  a.max_ctx = p->max_context;
  a.max_nodes = p->max_nodes;
  a.log_b = p->block_size == 16 ? 4 : p->block_size == 32 ? 5 : 6;
  a.groups = l.groups;
  a.units = l.units;
  a.nsplit = l.nsplit;
  a.chunk = l.chunk;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  char* ws = (char*)p->workspace;
  a.counters = (int*)ws;
  a.pm = (float*)(ws + l.pm);
  a.pl = (float*)(ws + l.pl);
  a.part = (float*)(ws + l.part);
  const dim3 grid((unsigned)((int64_t)l.units * l.nsplit));
  hipStream_t st = (hipStream_t)stream;
  if (p->head_dim == 64) {
    if (int8) hipLaunchKernelGGL((tree_attention_kernel<64, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((tree_attention_kernel<64, 0>), grid, dim3(256), 0, st, a);
  } else {
    if (int8) hipLaunchKernelGGL((tree_attention_kernel<128, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((tree_attention_kernel<128, 0>), grid, dim3(256), 0, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "tree attention launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}
