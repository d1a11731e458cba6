// Attention of drafted trees over the paged cache on the matrix cores (gfx950).
//
// A sequence's n nodes, each with G query heads for a KV head, make n G rows that read the same keys; row m is node m / G,
// head m % G, so that small trees fill whole 16-row tiles whatever the group size. A row sees the sequence's cached tokens
// and the nodes in its mask. The reference has no counterpart: it decodes one token per step.
//
// Work unit: (sequence, KV head, 64 or 128 rows); its keys are cut into splits of `chunk`, one workgroup each. The workgroup
// brings 128 or 64 keys at a time into LDS (registers ahead of them carry the next stages), each of its waves takes 16 rows:
//   S^T[16 keys x 16 rows] = K[16 x 32 d] . Q^T[32 d x 16 rows]   v_mfma_f32_16x16x32_bf16
//   hidden keys -> -inf; online softmax per row in the exp2 domain
//   O^T[16 d x 16 rows] += V^T . P^T
// INT8 pools: the codes go to LDS as bf16, exactly; the scores are multiplied by K's scales and the probabilities by V's in
// fp32. Splits write (m, l, O), all fp32, and the last of a unit's to arrive merges them.
// P enters the second product as two bf16 terms, 16 bits of it: one alone gives errors as large as the result's own rounding
// (2.3e-3 of it in all against 1.7e-3). The second is taken from p (1 + 2^-20), so that it is never zero against an infinite
// V.
//
// What bounds it: with few rows the pools' bytes (one node, 7 heads a KV head, 32 sequences of 8192 keys: 31 us, 4.4 TB/s);
// from about 16 nodes on the vector ALUs, which turn each score into two bf16 terms of p, and the wait of the waves for each
// other at a stage's end: a stage of 64 keys and 128 rows takes some 2400 cycles, 1000 of them the softmax of a SIMD's two
// waves, 460 the scores, 370 the second product. 16 nodes, 32 sequences of 8192 keys: 47 us of 27 for the bytes (INT8: 58 of
// 14); 64 nodes, 16 ragged sequences about 12000 long, head_dim 128: 152 us of 43; INT8, 11 nodes, 64 sequences of 4096,
// head_dim 128: 72 us of 28. Short calls take the chain of one workgroup's loads: 12 us for 5 nodes at 1024 keys.
#include <algorithm>
#include <type_traits>

#include "decode_common.h"

namespace sipa {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kTreeMaxSplits = 128;
constexpr int kTreeMaxChunk = 16384;  // block ids of a split in LDS: 4 KB
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
  int32_t nsplit, chunk;
  int32_t log_spread;      // a pair has 1 << log_spread XCDs
  float scale_log2;
  int* counters;           // [units]
  float* pm;               // [units][nsplit][rows of a group]
  float* pl;               // the same
  float* part;             // [units][nsplit][rows of a group][D]
};

// A scale as it lies in memory, and its value: apart, so that the load is waited for only where the value is needed.
__device__ __forceinline__ uint32_t scale_bits(const void* base, bool f32, int64_t i) {
  return f32 ? ((const uint32_t*)base)[i] : (uint32_t)((const uint16_t*)base)[i];
}

__device__ __forceinline__ float scale_value(uint32_t bits, bool f32) {
  return f32 ? __uint_as_float(bits) : f16_bits_to_f32(bits);
}

// Eight int8 codes (two words) as bf16, exactly.
__device__ __forceinline__ u32x4 tree_codes(uint32_t w0, uint32_t w1) {
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? w0 : w1;
    const int b = 16 * (i & 1);
    x[i] = pack_bf16x2((float)(int8_t)(w >> b), (float)(int8_t)(w >> (b + 8)));
  }
  return x;
}

// MR row tiles of 16 per wave, RW waves side by side over the rows, KW waves one after the other over the keys, each KPW
// keys of a stage of KW KPW; NPRE stages in flight in registers.
template <int D, int MODE, int MR, int RW, int KW, int KPW, int NPRE>
__global__ void __launch_bounds__(64 * RW * KW, 2) tree_attention_kernel(const TreeArgs a) {
  constexpr int KT = KW * KPW, MT = KPW / 16, HT = KPW / 32, P = D + 16, KS = D / 32, DT = D / 16;
  constexpr int PT = 64 * RW * KW, ROWS = 16 * MR * RW;
  constexpr int CH = MODE == 0 ? 8 : 16, CPK = D / CH, NCH = KT * CPK;  // 16-byte parts of a key, of a stage
  constexpr int LPT = (NCH + PT - 1) / PT, SPT = MODE == 0 ? 0 : (2 * KT + PT - 1) / PT;
  constexpr int TE = KT * P;
  __shared__ __align__(16) uint16_t sm[2][2][TE];  // [buffer][K, V][key][P]
  __shared__ __align__(16) float sscale[MODE == 0 ? 1 : 2][2][MODE == 0 ? 4 : KT];  // [buffer][K, V][key]
  __shared__ int bids[kTreeMaxChunk / 16];
  __shared__ uint64_t masks[ROWS * 4];  // [node of the group][word]
  __shared__ int last_flag, dirty;

  // Workgroup L is dealt to XCD L % 8: a pair's row groups and splits share one, so that its L2 serves the groups the same
  // keys and the merge its partials. With few pairs their splits go round 1 << a.log_spread XCDs.
  // The heads' sequences are shifted against each other, so that no XCD has the same long sequence twice (4 sequences of up to
  // 128 nodes x 15000 keys, INT8: 97 -> 86 us).
  const int L = blockIdx.x, log_side = 3 - a.log_spread;  // 1 << log_side pairs side by side
  const int per = ((a.nsplit + (1 << a.log_spread) - 1) >> a.log_spread) * a.groups, turn = (L >> 3) / per, in = (L >> 3) - turn * per;
  const int pair = (L & ((1 << log_side) - 1)) + (turn << log_side), sp = ((in / a.groups) << a.log_spread) + ((L & 7) >> log_side);
  if (pair >= a.S * a.Hkv || sp >= a.nsplit) return;  // the grid is padded
  const int rg = in % a.groups, h = pair / a.S, s = (pair + 3 * h) % a.S;
  const int u = pair * a.groups + rg;
  const int row0 = a.qs[s], all = a.qs[s + 1] - row0, n = min(min(all, a.max_nodes), a.T - row0);
  const int G = a.G, M = n * G, m0 = rg * ROWS;
  if (n <= 0 || row0 < 0 || m0 >= M) return;
  const int ctx = min(a.ctx[s], a.max_ctx), start = ctx - all;
  const int nvalid = max(1, (ctx + a.chunk - 1) / a.chunk);
  if (sp >= nvalid) return;
  const int k_lo = sp * a.chunk, k_hi = min(k_lo + a.chunk, ctx);
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave / RW;
  // odd key waves take the rows in reverse: a last row tile that is missing then costs each SIMD alike
  const int rw = kw & 1 ? RW - 1 - wave % RW : wave % RW;

  const int nkeys = max(k_hi - k_lo, 0), first_col = k_lo >> a.log_b;
  const int32_t* table = a.bt + (int64_t)s * a.bt_ss;
  for (int i = tid; i << a.log_b < nkeys; i += PT) bids[i] = min(max(table[min(first_col + i, a.bt_w - 1)], 0), a.nb - 1);

  const int node0 = m0 / G, nodes = min((m0 + ROWS - 1) / G, n - 1) - node0 + 1;  // the group's nodes, at most ROWS
  for (int i = tid; i < nodes * a.words; i += PT) masks[i] = a.masks[(int64_t)(row0 + node0) * a.words + i];
  if (tid == 0) dirty = 0;
  int node[MR], head[MR];
  bool tile_valid[MR];  // wave-uniform
  bf16x8 qop[MR][KS];
#pragma unroll
  for (int c = 0; c < MR; ++c) {
    const int m = m0 + 16 * (MR * rw + c) + r, at = min(m, M - 1);
    tile_valid[c] = m0 + 16 * (MR * rw + c) < M;
    node[c] = at / G;
    head[c] = at - node[c] * G;
#pragma unroll
    for (int j = 0; j < KS; ++j)
      qop[c][j] = __builtin_bit_cast(bf16x8, *(const u32x4*)(a.q + (int64_t)(row0 + node[c]) * a.q_st +
                                                             (int64_t)(h * G + head[c]) * a.q_sh + 32 * j + 8 * q4));
  }
  constexpr float kSlack = 8.f, kFastRange = 16.f;
  const float inv_scale_log2 = MODE == 0 ? 1.f / a.scale_log2 : 1.f;
  float m_run[MR], m_off[MR], fast_thr[MR];  // m_off: m_run, or 0 while that is -inf
  f32x4 l_run[MR];  // MODE 0: an accumulator whose every row holds the sum; MODE 1: a lane's own four sums
  f32x4 acc[MR][DT];
#pragma unroll
  for (int c = 0; c < MR; ++c) {
    m_run[c] = fast_thr[c] = kNegInf, m_off[c] = 0.f, l_run[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[c][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int tr_off = tr16_offset(r, q4, P);
  bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
  asm volatile("" : "+v"(ones));  // kept in registers
  __syncthreads();  // block ids

  const int ntiles = (nkeys + KT - 1) / KT;
  u32x4 rk[NPRE][LPT], rv[NPRE][LPT];
  uint32_t rs[NPRE][SPT ? SPT : 1];
  // A thread's parts of a stage keep their place in their blocks from stage to stage (a stage is whole blocks): what changes
  // is the block id. Keys past the split's end are read too, inside its last block; they are hidden, and cleaned below.
  const int es = MODE == 0 ? 2 : 1, last_id = max((nkeys - 1) >> a.log_b, 0);
  const uint32_t kv_bytes = (uint32_t)a.kv_sn * es;  // of a block (host-checked)
  const uint8_t* kbase[LPT];
  const uint8_t* vbase[LPT];
  int part_id[LPT];
#pragma unroll
  for (int i = 0; i < LPT; ++i) {
    const int c = tid + PT * i, key = c / CPK;
    const int64_t e = ((int64_t)h * a.kv_sh + (key & ((1 << a.log_b) - 1)) * D + CH * (c % CPK)) * es;
    kbase[i] = (const uint8_t*)a.k + e;
    vbase[i] = (const uint8_t*)a.v + e;
    part_id[i] = key >> a.log_b;
  }
  auto gload = [&](int set, int t) {
#pragma unroll
    for (int i = 0; i < LPT; ++i) {
      if (NCH % PT != 0 && tid + PT * i >= NCH) break;
      const uint64_t at = (uint64_t)(uint32_t)bids[min((KT * t >> a.log_b) + part_id[i], last_id)] * kv_bytes;
      rk[set][i] = *(const u32x4*)(kbase[i] + at);
      rv[set][i] = *(const u32x4*)(vbase[i] + at);
    }
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const int c = tid + PT * i;
      if (2 * KT % PT != 0 && c >= 2 * KT) break;
      const int key = c % KT, off = key & ((1 << a.log_b) - 1);
      const int64_t blk = bids[min((KT * t >> a.log_b) + (key >> a.log_b), last_id)];
      rs[set][i] = c < KT ? scale_bits(a.ks, a.ks_f32, (int64_t)h * a.ks_sh + blk * a.ks_sn + off)
                          : scale_bits(a.vs, a.vs_f32, (int64_t)h * a.vs_sh + blk * a.vs_sn + off);
    }
  };
  // Infinities and NaN among the nodes' V: a row that does not see them must not take 0 * V into its sums. They go to LDS
  // as zeros, and the rows that see them take them up at the end.
  auto cleaned = [&](u32x4 v, int key) {
    if (key < start) return v;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t keep = ((v[w] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((v[w] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
      if (keep != 0xffffffffu && key < k_hi) dirty = 1;
      v[w] &= keep;
    }
    return v;
  };
  auto sstore = [&](int set, int t) {
    const int buf = t & 1;
    const bool check = k_lo + KT * (t + 1) > start;  // uniform: some key of the stage is a node
#pragma unroll
    for (int i = 0; i < LPT; ++i) {
      const int c = tid + PT * i;
      if (NCH % PT != 0 && c >= NCH) break;
      const int e = (c / CPK) * P + CH * (c % CPK);
      if constexpr (MODE == 0) {
        *(u32x4*)(&sm[buf][0][e]) = rk[set][i];
        *(u32x4*)(&sm[buf][1][e]) = check ? cleaned(rv[set][i], k_lo + KT * t + c / CPK) : rv[set][i];
      } else {
        // At head_dim 64 odd lanes store their second half first, as 16 bytes of each 32 use half the banks (24 nodes, 24 ragged
        // sequences about 6000 long: 119 -> 97 us, and 148 registers for 244); at 128 it loses 1 % (72.3 -> 72.9).
        const int odd = D == 64 ? tid & 1 : 0;
        const u32x4 k = rk[set][i], v = rv[set][i];
        *(u32x4*)(&sm[buf][0][e + 8 * odd]) = tree_codes(odd ? k[2] : k[0], odd ? k[3] : k[1]);
        *(u32x4*)(&sm[buf][0][e + 8 - 8 * odd]) = tree_codes(odd ? k[0] : k[2], odd ? k[1] : k[3]);
        *(u32x4*)(&sm[buf][1][e + 8 * odd]) = tree_codes(odd ? v[2] : v[0], odd ? v[3] : v[1]);
        *(u32x4*)(&sm[buf][1][e + 8 - 8 * odd]) = tree_codes(odd ? v[0] : v[2], odd ? v[1] : v[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const int c = tid + PT * i;
      if (2 * KT % PT != 0 && c >= 2 * KT) break;
      sscale[buf][c / KT][c % KT] = c < KT ? scale_value(rs[set][i], a.ks_f32) * a.scale_log2 : scale_value(rs[set][i], a.vs_f32);
    }
  };
  // Which of the keys x0 .. x0 + KPW - 1 the row of a node sees, key x0 + b in bit b.
  auto sees = [&](int nd, int x0) {
    const int rel = x0 - start, shift = rel & 63;
    auto word = [&](int w) {
      const uint64_t x = masks[(nd - node0) * a.words + min(max(w, 0), a.words - 1)];
      return w < 0 ? ~0ull : w < a.words ? x : 0ull;
    };
    uint64_t bits = word(rel >> 6) >> shift;
    if (shift) bits |= word((rel >> 6) + 1) << (64 - shift);
    return k_hi - x0 >= 64 ? bits : bits & ((1ull << (k_hi - x0)) - 1);
  };
  auto tile = [&](int t) {
    const int x0 = k_lo + KT * t + KPW * kw;  // the wave's first key
    if (x0 >= k_hi || !tile_valid[0]) return;  // wave-uniform
    const int buf = t & 1;
    const uint16_t* sk = sm[buf][0] + KPW * kw * P;
    const uint16_t* sv = sm[buf][1] + KPW * kw * P;
    const bool masked = x0 + KPW > min(start, k_hi);  // some key is a node, or past the split's end
    bf16x8 kop[MT][KS];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < KS; ++j) kop[mt][j] = *(const bf16x8*)(sk + (16 * mt + r) * P + 32 * j + 8 * q4);
    u32x4 hi[MR][HT], lo[MR][HT];  // bf16 pairs
#pragma unroll
    for (int c = 0; c < MR; ++c) {
      f32x4 sc[MT];  // row (mt, q4, i) holds key 16 mt + 4 q4 + i
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KS; ++j) sc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[mt][j], qop[c][j], sc[mt], 0, 0, 0);
        if constexpr (MODE == 1) sc[mt] *= *(const f32x4*)(sscale[buf][0] + KPW * kw + 16 * mt + 4 * q4);  // log2 units
      }
      if (masked) {
        const uint64_t bits = sees(node[c], x0) >> (4 * q4);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(bits >> (16 * mt + i) & 1)) sc[mt][i] = kNegInf;
      }
      // Each lane's largest score. The row's max (two cross-lane steps more) is looked at only when some score exceeds the
      // running one by more than 2^kFastRange, and raised only past 2^kSlack: p stays far inside fp32 otherwise.
      float mx = sc[0][0];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = vmax(mx, sc[mt][i]);
      if (__builtin_amdgcn_ballot_w64(mx > fast_thr[c])) {
        mx = max_over_rows_swap(mx) * (MODE == 0 ? a.scale_log2 : 1.f);
        if (__builtin_amdgcn_ballot_w64(mx > m_run[c] + kSlack)) {
          const float m_new = fmaxf(m_run[c], mx);
          const float alpha = fast_exp2(m_run[c] - (m_new == kNegInf ? 0.f : m_new));  // 0 while the row has seen no key
          l_run[c] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[c][dt] *= alpha;
          m_run[c] = m_new;
          m_off[c] = m_new == kNegInf ? 0.f : m_new;
          fast_thr[c] = (m_new + kFastRange) * inv_scale_log2;
        }
      }
#pragma unroll
      for (int hf = 0; hf < HT; ++hf) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = sc[2 * hf + (i >> 2)][i & 3];
          p[i] = fast_exp2(MODE == 0 ? fmaf(x, a.scale_log2, -m_off[c]) : x - m_off[c]);
        }
        if constexpr (MODE == 1) {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const f32x4 vs = *(const f32x4*)(sscale[buf][1] + KPW * kw + 32 * hf + 4 * i + 4 * q4);
#pragma unroll
            for (int x = 0; x < 4; ++x) l_run[c][x] += p[i + x];
            if (masked) {
#pragma unroll
              for (int x = 0; x < 4; ++x) p[i + x] = p[i + x] == 0.f ? 0.f : p[i + x] * vs[x];  // a hidden scale may be anything
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) p[i + x] *= vs[x];
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          uint32_t cut[2];
          float rest[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            cut[x] = __float_as_uint(p[i + x]) & 0xffff0000u;
            rest[x] = fmaf(p[i + x], 1.f + 0x1p-20f, -__uint_as_float(cut[x]));
          }
          hi[c][hf][i >> 1] = __builtin_amdgcn_perm(cut[1], cut[0], 0x07060302u);
          lo[c][hf][i >> 1] = pack_bf16x2(rest[0], rest[1]);
        }
        if constexpr (MODE == 0) {  // the sums on the matrix cores, of the values that the product uses
          l_run[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, hi[c][hf]), l_run[c], 0, 0, 0);
          l_run[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, lo[c][hf]), l_run[c], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int hf = 0; hf < HT; ++hf)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 vop = read_v_operand<bf16x8>(sv + 32 * P * hf, tr_off, P, 16 * dt);
#pragma unroll
        for (int c = 0; c < MR; ++c) {
          acc[c][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, __builtin_bit_cast(bf16x8, hi[c][hf]), acc[c][dt], 0, 0, 0);
          acc[c][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, __builtin_bit_cast(bf16x8, lo[c][hf]), acc[c][dt], 0, 0, 0);
        }
      }
  };
  if (ntiles > 0) {
#pragma unroll
    for (int k = 0; k < NPRE; ++k) {
      gload(k, k);
      asm volatile("" ::: "memory");  // in this order
    }
    sstore(0, 0);
    __syncthreads();
    // register set k % NPRE carries stage k to its LDS store; loads past the last stage read its last key again, so that
    // every wait is for a fixed count, and stages past it compute nothing
    for (int tb = 0; tb < ntiles; tb += NPRE) {
#pragma unroll
      for (int k = 0; k < NPRE; ++k) {
        const int t = tb + k;
        gload(k, t + NPRE);
        tile(t);
        sstore((k + 1) % NPRE, t + 1);  // that buffer was last read before the last barrier
        __syncthreads();
      }
    }
  }
  float l[MR];
#pragma unroll
  for (int c = 0; c < MR; ++c) {
    l[c] = MODE == 0 ? l_run[c][0] : sum_over_rows_swap(l_run[c][0] + l_run[c][1] + l_run[c][2] + l_run[c][3]);
    if (l[c] != l[c]) m_run[c] = 0.f;  // NaN scores never raise the max: the merges see the row by its sum
  }
  if constexpr (KW > 1) {
    // The key waves' states join in LDS (the tile buffers are free after the last barrier): waves kw > 0 leave theirs,
    // wave kw = 0 of the same rows takes them up one after the other.
    constexpr int XS = DT * 4 + 4;  // floats of a lane: O, m, l
    static_assert((KW - 1) * RW * MR * 64 * XS * 4 <= (int)sizeof(sm), "the states fit the tile buffers");
    float* xs = (float*)&sm[0][0][0];
    if (kw > 0) {
#pragma unroll
      for (int c = 0; c < MR; ++c) {
        float* x = xs + ((((kw - 1) * RW + rw) * MR + c) * 64 + lane) * XS;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *(f32x4*)(x + 4 * dt) = acc[c][dt];
        x[4 * DT] = m_run[c];
        x[4 * DT + 1] = l[c];
      }
    }
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int k = 1; k < KW; ++k)
#pragma unroll
        for (int c = 0; c < MR; ++c) {
          const float* x = xs + ((((k - 1) * RW + rw) * MR + c) * 64 + lane) * XS;
          const float m1 = x[4 * DT], l1 = x[4 * DT + 1];
          const float top = vmax(m_run[c], m1);
          if (top == kNegInf) continue;
          const float f0 = fast_exp2(m_run[c] - top), f1 = fast_exp2(m1 - top);
          l[c] = f0 * l[c] + f1 * l1;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[c][dt] = f0 * acc[c][dt] + f1 * *(const f32x4*)(x + 4 * dt);
          m_run[c] = top;
        }
    }
  }
  const bool owner = kw == 0;
  if (MODE == 0 && dirty && owner) {  // (set before the loop's last barrier)
    for (int key = max(start, k_lo); key < k_hi; ++key) {
      const uint16_t* v = (const uint16_t*)a.v + (int64_t)h * a.kv_sh + (int64_t)bids[(key >> a.log_b) - first_col] * a.kv_sn +
                          (int64_t)(key & ((1 << a.log_b) - 1)) * D + 4 * q4;
#pragma unroll
      for (int c = 0; c < MR; ++c) {
        const bool on = sees(node[c], key) & 1;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = bf16_bits_to_f32(v[16 * dt + i]);
            if (on && !(fabsf(x) < __builtin_huge_valf())) acc[c][dt][i] += x;
          }
      }
    }
  }
  if (nvalid == 1) {
    if (!owner) return;
#pragma unroll
    for (int c = 0; c < MR; ++c) {
      if (m0 + 16 * (MR * rw + c) + r >= M) continue;
      const float inv = l[c] == 0.f ? 0.f : 1.f / l[c];  // no key: zeros
      uint16_t* o = a.out + (int64_t)(row0 + node[c]) * a.o_st + (int64_t)(h * G + head[c]) * a.o_sh + 4 * q4;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *(u32x2*)(o + 16 * dt) = u32x2{pack_bf16x2(acc[c][dt][0] * inv, acc[c][dt][1] * inv),
                                       pack_bf16x2(acc[c][dt][2] * inv, acc[c][dt][3] * inv)};
    }
    return;
  }
  // The split's state: m, l and O of each row, as the accumulators hold them. (O / l in fp16 takes half the bytes, but holds no
  // V under 2^-25, and one exponent a row no finite value beside an infinite one.)
  const int64_t first = (int64_t)u * a.nsplit * ROWS;
  const int split_bytes = ROWS * D * 4;
  const __amdgpu_buffer_rsrc_t rows =
      __builtin_amdgcn_make_buffer_rsrc(a.part + first * D, (short)0, a.nsplit * split_bytes, 0x00020000);
  if (owner) {
#pragma unroll
    for (int c = 0; c < MR; ++c) {
      const int slot = 16 * (MR * rw + c) + r;
      if (m0 + slot >= M) continue;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[c][dt]), rows,
                                               sp * split_bytes + (slot * D + 16 * dt + 4 * q4) * 4, 0, kAuxSc1);
      if (q4 == 0) {
        store_coherent(a.pm + first + sp * ROWS + slot, m_run[c]);
        store_coherent(a.pl + first + sp * ROWS + slot, l[c]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    // +2^16 from a workgroup that is not on the pair's one XCD: the last to arrive then reads through memory, else from its L2
    uint32_t xcc;
    asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(xcc));
    const int away = a.log_spread > 0 || (int)(xcc & 0xf) != (L & 7);
    const int prev = __hip_atomic_fetch_add(a.counters + u, 1 + (away << 16), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_flag = (prev & 0xffff) == nvalid - 1 ? 1 + ((prev >> 16) + away == 0) : 0;
  }
  __syncthreads();
  if (!last_flag) return;
  const __amdgpu_buffer_rsrc_t mrows =
      __builtin_amdgcn_make_buffer_rsrc(a.pm + first, (short)0, a.nsplit * ROWS * 4, 0x00020000);
  const __amdgpu_buffer_rsrc_t lrows =
      __builtin_amdgcn_make_buffer_rsrc(a.pl + first, (short)0, a.nsplit * ROWS * 4, 0x00020000);
  // Every split's m and l first, in LDS, then each thread 8 channels of a row with kMerge splits' loads in flight.
  float* lm = (float*)&sm[0][0][0];  // [nvalid][ROWS] m, then l
  float* ll = lm + nvalid * ROWS;
  auto merge = [&](auto tag) {
    constexpr int AUX = decltype(tag)::value, kMerge = 8;
    for (int i = tid; i < nvalid * ROWS; i += PT) {
      lm[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(mrows, i * 4, 0, AUX));
      ll[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(lrows, i * 4, 0, AUX));
    }
    __syncthreads();
    for (int i = tid; i < ROWS * (D / 8); i += PT) {
      const int slot = i / (D / 8), ch = 8 * (i % (D / 8));
      if (m0 + slot >= M) break;
      float top = kNegInf, den = 0.f;
      for (int j = 0; j < nvalid; ++j) top = fmaxf(top, lm[j * ROWS + slot]);
      f32x4 num[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      for (int j0 = 0; j0 < nvalid; j0 += kMerge) {
        f32x4 o[kMerge][2];
#pragma unroll
        for (int x = 0; x < kMerge; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            o[x][y] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                rows, min(j0 + x, nvalid - 1) * split_bytes + (slot * D + ch + 4 * y) * 4, 0, AUX));
#pragma unroll
        for (int x = 0; x < kMerge; ++x) {
          const int j = min(j0 + x, nvalid - 1);
          const float f = j0 + x >= nvalid || top == kNegInf ? 0.f : fast_exp2(lm[j * ROWS + slot] - top);
          const float w = f * ll[j * ROWS + slot];
          if (w == 0.f) continue;  // a split without a key for the row
          den += w;
#pragma unroll
          for (int y = 0; y < 2; ++y) num[y] += f * o[x][y];
        }
      }
      const float inv = den == 0.f ? 0.f : 1.f / den;
      const int nd = (m0 + slot) / G, hd = (m0 + slot) - nd * G;
      *(u32x4*)(a.out + (int64_t)(row0 + nd) * a.o_st + (int64_t)(h * G + hd) * a.o_sh + ch) =
          u32x4{pack_bf16x2(num[0][0] * inv, num[0][1] * inv), pack_bf16x2(num[0][2] * inv, num[0][3] * inv),
                pack_bf16x2(num[1][0] * inv, num[1][1] * inv), pack_bf16x2(num[1][2] * inv, num[1][3] * inv)};
    }
  };
  if (last_flag == 2) {
    asm volatile("buffer_inv sc0" ::: "memory");  // sc0 loads may hit the CU's L1: drop any earlier copy first
    merge(std::integral_constant<int, kAuxSc0>());
  } else {
    merge(std::integral_constant<int, kAuxSc1>());
  }
  if (tid == 0) __hip_atomic_store(a.counters + u, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace sipa

using namespace sipa;

struct TreeLayout {
  int variant, rows;  // index into the launch table below, rows of a workgroup
  int groups, units, nsplit, chunk, log_spread;
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

struct TreeVariant {
  int mr, rw, kw, kpw;
};
constexpr TreeVariant kTreeVariants[] = {{1, 4, 2, 64}, {1, 8, 1, 64}};  // up to 64 rows, more

// Bytes of the kernel's tile buffers, which the merge's m and l have to fit: the number of splits, and with it the context, is
// limited by them (40 splits, 655360 keys, for more than 64 rows at head_dim 64).
static int tree_tile_bytes(const TreeVariant& v, int D) { return 2 * 2 * v.kw * v.kpw * (D + 16) * 2; }

// XCDs that a pair's splits go round, as a power of two. Few pairs on one XCD each would leave CUs idle (one sequence of 2 KV
// heads has 64 of 256); against that, the merge then reads through memory. Times against one XCD a pair, in the mean: 2 pairs
// (48 batches) 0.86 on two XCDs, 0.815 on four, 0.81 on eight (contexts over 10000 keys and several row groups 0.57, up to 3000
// no gain or up to 1.24), so one pair, which has half their CUs, goes round all eight; 3 and 4 pairs (29 batches) 0.97; 5 to 16
// pairs (320 batches) 1.00 to 1.05; 17 to 64 (71) 1.02 to 1.20.
static int tree_log_spread(int64_t pairs, int nsplit) {
  const int want = pairs == 1 ? 3 : pairs == 2 ? 2 : pairs <= 4 ? 1 : 0;
  return nsplit == 1 ? 0 : want;
}

// The number of splits: the cheapest by a count of keys. A workgroup costs its split's keys and 256 more (its start and end), a
// CU takes one after the other, two at once where both fit (the larger variant over plain pools at head_dim 64: 1.6 times one's
// time), and a merge costs 256 keys and 24 a split. The call is not given the lengths: the count takes every sequence for one of
// max_context keys; where the trees' sizes differ (the token count shows it) many workgroups find no rows or keys, and half of
// the count is that of 0.7 of the workgroups. Over 508 batches (1 to 128 sequences, 1 to 128 nodes, contexts to 16384 keys, both
// types and head sizes, over half ragged) it takes 3.6 % over the best count's time in the mean, 1.39 times at most. One
// workgroup per CU, rounded up, takes 15 % in the mean, 2.4 times at most: 40 sequences of 2 heads make 320 workgroups of 4
// splits each (36 us for 6 nodes at 3000 keys, 16-bit pools, head_dim 64), where 3 splits fill 240 of the 256 CUs (23 us).
static int tree_splits(const sipa_tree_params* p, int groups, int kt, bool two, int cus, int most) {
  const int64_t pairs = (int64_t)p->num_seqs * p->num_kv_heads, per_xcd = std::max(cus / 8, 1);
  const bool differ = p->num_tokens < (int64_t)p->num_seqs * p->max_nodes;
  auto fifths = [&](int64_t wgs) {  // of a lone workgroup's time, for the workgroups of an XCD
    const int64_t turns = (wgs + per_xcd - 1) / per_xcd;
    return two ? 8 * (turns / 2) + 5 * (turns % 2) : 5 * turns;
  };
  int best = 1;
  int64_t least = INT64_MAX;
  for (int n = 1; n <= most && (int64_t)128 * (n - 1) < p->max_context; n += 1 + n / 8) {
    const int64_t chunk = ((p->max_context + n - 1) / n + kt - 1) / kt * kt;
    const int spread = 1 << tree_log_spread(pairs, n), side = 8 / spread;
    const int64_t wgs = (pairs + side - 1) / side * groups * ((n + spread - 1) / spread);
    const int64_t time = fifths(wgs) + fifths(differ ? (7 * wgs + 9) / 10 : wgs);
    const int64_t cost = time * (chunk + 256) + 10 * (n > 1 ? 256 + 24 * n : 0);
    if (cost < least) least = cost, best = n;
  }
  return best;
}

static int tree_layout(const sipa_tree_params* p, TreeLayout* l) {
  const int G = p->num_q_heads / p->num_kv_heads;
  const int need = p->max_nodes * G;
  l->variant = need <= 64 ? 0 : 1;
  const TreeVariant& v = kTreeVariants[l->variant];
  l->rows = 16 * v.mr * v.rw;
  l->groups = (need + l->rows - 1) / l->rows;
  const int64_t units = (int64_t)p->num_seqs * p->num_kv_heads * l->groups;
  SIPA_CHECK(units <= 0x7fffffff / kTreeMaxSplits, SIPA_EINVAL, "%lld units exceed the grid limit", (long long)units);
  l->units = (int)units;
  const int kt = v.kw * v.kpw;  // whole stages
  const int most = std::min(kTreeMaxSplits, tree_tile_bytes(v, p->head_dim) / (8 * l->rows));
  int splits = std::min(p->num_splits, most);
  if (splits <= 0) {
    const int cus = sipa_device_cu_count(-1);
    if (cus < 0) return cus;
    splits = tree_splits(p, l->groups, kt, l->variant == 1 && p->head_dim == 64 && p->kv_mode == SIPA_KV_PLAIN, cus, most);
  }
  const int chunk = (p->max_context + splits - 1) / splits;
  l->chunk = std::min((chunk + kt - 1) / kt * kt, kTreeMaxChunk);
  l->nsplit = (p->max_context + l->chunk - 1) / l->chunk;
  SIPA_CHECK(l->nsplit <= most, SIPA_EUNSUPPORTED, "max_context %d past %d splits of %d keys", p->max_context, most, kTreeMaxChunk);
  l->log_spread = tree_log_spread((int64_t)p->num_seqs * p->num_kv_heads, l->nsplit);
  l->pm = l->pl = l->part = l->total = 0;
  if (l->nsplit > 1) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t rows = units * l->nsplit * l->rows;
    SIPA_CHECK((int64_t)l->nsplit * l->rows * p->head_dim * 4 <= 0x7fffffff, SIPA_EINVAL, "split state too large");
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

template <int D, int MODE, int V>
static void launch_variant(dim3 grid, hipStream_t st, const TreeArgs& a) {
  constexpr TreeVariant v = kTreeVariants[V];
  hipLaunchKernelGGL((tree_attention_kernel<D, MODE, v.mr, v.rw, v.kw, v.kpw, D == 64 ? 4 : 3>), grid, dim3(64 * v.rw * v.kw), 0, st, a);
}

template <int D, int MODE>
static void launch_tree(int variant, dim3 grid, hipStream_t st, const TreeArgs& a) {
  if (variant == 0) launch_variant<D, MODE, 0>(grid, st, a);
  else launch_variant<D, MODE, 1>(grid, st, a);
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
  SIPA_CHECK(p->kv_stride_n >= 0 && p->kv_stride_n <= 0x7fffffff, SIPA_EUNSUPPORTED, "blocks %lld elements apart",
             (long long)p->kv_stride_n);
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
  a.nsplit = l.nsplit;
  a.log_spread = l.log_spread;
  a.chunk = l.chunk;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  char* ws = (char*)p->workspace;
  a.counters = (int*)ws;
  a.pm = (float*)(ws + l.pm);
  a.pl = (float*)(ws + l.pl);
  a.part = (float*)(ws + l.part);
  const int64_t side = 8 >> l.log_spread, rounds = ((int64_t)p->num_seqs * p->num_kv_heads + side - 1) / side;
  const dim3 grid((unsigned)(8 * rounds * l.groups * ((l.nsplit + (1 << l.log_spread) - 1) >> l.log_spread)));
  hipStream_t st = (hipStream_t)stream;
  if (p->head_dim == 64) {
    if (int8) launch_tree<64, 1>(l.variant, grid, st, a);
    else launch_tree<64, 0>(l.variant, grid, st, a);
  } else {
    if (int8) launch_tree<128, 1>(l.variant, grid, st, a);
    else launch_tree<128, 0>(l.variant, grid, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "tree attention launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}
