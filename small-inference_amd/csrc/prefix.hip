// Decode attention of sequences whose block tables begin with the same blocks (gfx950): the shared keys are read once for a
// whole group of them. The reference reads every sequence's context by itself.
//
// One token a sequence. A row (sequence, query head) splits its softmax over the keys of its group's prefix and those of its
// own: (m, l, O) of each part, m the part's largest score, l = sum 2^(s - m), O = sum 2^(s - m) v, joined as
//   M = max m,  out = sum 2^(m - M) O / sum 2^(m - M) l.
// Prefix items: (group, KV head, up to ROWS of the group's rows, keys), a workgroup each: the members' G query heads make one
// matrix of rows that see every key, so the product has full tiles whatever G is. Own pieces: (sequence, KV head, keys), G rows
// of 16, a wave each, eight to a workgroup: most are short, and a wave needs no other. Both kinds are in one launch, so that the
// pieces' loads run beside the items' products; a second, small one joins a row's parts.
//
// A row is in one group: of prefixes within prefixes the plan's caller chooses one level, the others' keys are read for every row.
//
// What bounds it: with long contexts of their own the pools' bytes (256 sequences behind 2048 tokens with about 600 of their own,
// head_dim 128, 16-bit pools: 49 us with pools that change from call to call, 32 of them for the bytes at a copy's rate, and 40 with
// pools that stay in the caches; read apart 93); with long prefixes and many rows the vector ALUs and LDS reads of the items, and
// tiles that are not full (2 x 37 sequences at 30016 tokens: 35 us, 5.7 for the products; each group's 259 rows make two tiles of
// 128 and one of 3); INT8 the conversion of codes; short batches the round trips of two launches, 9 us.
#include <algorithm>

#include "decode_common.h"

namespace sipa {

constexpr int kPrefixMaxChunk = 16384;  // keys of a prefix item: its block ids stand in LDS
constexpr int kPrefixThreads = 512, kPrefixWaves = 8;
constexpr int kPrefixStage = 64;  // keys in LDS at a time

struct PrefixArgs {
  const uint16_t* q;
  int64_t q_ss, q_sh;
  const void* k;
  const void* v;
  int64_t kv_sh, kv_sn;
  const int32_t* bt;
  int64_t bt_ss;
  int32_t bt_w;
  const int32_t* ctx;
  uint16_t* out;
  int64_t o_ss, o_sh;
  const void* ks;
  const void* vs;
  bool ks_f32, vs_f32;
  int64_t ks_sh, ks_sn, vs_sh, vs_sn;
  // The plan. Items: table row, first member, rows, first row, KV head, first key, end, state. Pieces: batch row, KV head, which
  // of the row's, how many those are, prefix tokens, state, -, -. Rows: prefix tokens, first row in the group, first state,
  // splits, row tiles, first piece's state, pieces of a KV head, -. Members: batch rows of the groups, one group after the other.
  const int32_t* items;    // [num_items][8]
  const int32_t* pieces;   // [num_pieces][8]
  const int32_t* rows;     // [S][8]
  const int32_t* members;  // [num_members]
  int32_t num_items, num_pieces, num_members, S, Hkv, G, nb, max_ctx;
  int32_t log_b;           // blocks of 1 << log_b tokens
  int32_t tile_rows;       // rows of a prefix item
  float scale_log2;
  // States, of the items' rows, then of the pieces': O, and (m, l).
  float* st_o;             // [num_items tile_rows + num_pieces G][D]
  float2* st_ml;
};

// Stores of states, in device memory: the two paths' would else be joined into flat ones, which also look for LDS.
typedef __attribute__((address_space(1))) f32x4 GlobalF32x4;
typedef __attribute__((address_space(1))) uint64_t GlobalU64;

// A sequence's keys: the prefix's `shared` (read with its group, or 0), then up to `planned` pieces of `chunk` keys of its own. A
// context that is shorter than its group's prefix is read by itself, from its first key on.
struct OwnKeys {
  int shared, ctx, chunk, pieces;
};

__device__ __forceinline__ OwnKeys own_keys(const PrefixArgs& a, int s, int tokens, int planned) {
  OwnKeys k;
  k.ctx = min(max(a.ctx[s], 0), a.max_ctx);
  k.shared = k.ctx >= tokens ? tokens : 0;
  const int own = k.ctx - k.shared;
  k.chunk = max(((own + planned - 1) / planned + 31) & ~31, 32);
  k.pieces = (own + k.chunk - 1) / k.chunk;
  return k;
}

// The four scales of consecutive keys, at any alignment, as they lie in memory, and their values: apart, so that the loads are
// waited for only where the values are needed. (fp16 scales: both halves are the same eight bytes.)
__device__ __forceinline__ u32x4 load_scales(const void* base, bool f32, int64_t i) {
  struct __attribute__((packed, aligned(2))) Eight {
    uint32_t w[2];
  };
  const char* at = (const char*)base + i * (f32 ? 4 : 2);
  const Eight lo = *(const Eight*)at, hi = *(const Eight*)(at + (f32 ? 8 : 0));
  return u32x4{lo.w[0], lo.w[1], hi.w[0], hi.w[1]};
}

__device__ __forceinline__ f32x4 four_scales(u32x4 s, bool f32) {
  const f32x4 half = {f16_bits_to_f32(s[0] & 0xffff), f16_bits_to_f32(s[0] >> 16), f16_bits_to_f32(s[1] & 0xffff),
                      f16_bits_to_f32(s[1] >> 16)};
  return f32 ? __builtin_bit_cast(f32x4, s) : half;
}

// One scale, by halves (of fp16 both are the same): loads under a branch of the type would be waited for at its end.
__device__ __forceinline__ u32x2 load_scale(const void* base, bool f32, int64_t i) {
  const uint16_t* at = (const uint16_t*)base + (f32 ? 2 * i : i);
  return u32x2{at[0], at[f32 ? 1 : 0]};
}

__device__ __forceinline__ float one_scale(u32x2 s, bool f32) {
  return f32 ? __uint_as_float(s[0] | s[1] << 16) : f16_bits_to_f32(s[0]);
}

// The softmax state of 16 rows in a wave, lane (r, q4) holding row r: O^T in the accumulators' layout (channels 16 dt + 4 q4 + i).
template <int D>
struct RowState {
  static constexpr int DT = D / 16;
  float m, off, threshold;  // off: m, or 0 while that is -inf
  f32x4 l;
  f32x4 acc[DT];

  __device__ __forceinline__ void clear() {
    m = threshold = kNegInf, off = 0.f, l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Takes up N keys' scores (hidden ones -inf), N a multiple of 32, score (mt, i) that of key 16 mt + 4 q4 + i: raises the
  // running max where one exceeds it by more than 2^16 (p stays far inside fp32), and returns the probabilities as two bf16
  // terms, 16 bits of them: one alone gives errors as large as the result's own rounding. The second is taken from
  // p (1 + 2^-20), so that it is never zero against an infinite V. What is left off is under 2^-15 of p (and the 2^-20, which the
  // sums take too in MODE 0), 2^-8 is the result's rounding. The decode kernel has as many bits over 16-bit blocks of 16 tokens
  // and 24 over larger blocks: of 1000 results 3 to 6 are neighbours of its own in either case, and the error against 64 bits is
  // the same to five digits (1.67e-3 of the norm); over INT8 blocks of 16 tokens, where it takes fp16 weights, 100 of 1000 and a
  // little less. MODE 0: raw scores; MODE 1: scores in log2 units, with V's scales at vs, and l takes the unscaled p.
  template <int MODE, int N>
  __device__ __forceinline__ void add(const f32x4 (&sc)[N / 16], float scale_log2, float inv_scale_log2, bf16x8 ones,
                                      const f32x4* vs, u32x4 (&hi)[N / 32], u32x4 (&lo)[N / 32]) {
    constexpr float kSlack = 8.f, kFastRange = 16.f;
    float mx = sc[0][0];
#pragma unroll
    for (int mt = 0; mt < N / 16; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = vmax(mx, sc[mt][i]);
    if (__builtin_amdgcn_ballot_w64(mx > threshold)) {
      mx = max_over_rows_swap(mx) * (MODE == 0 ? scale_log2 : 1.f);
      if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {
        const float m_new = fmaxf(m, mx);
        const float alpha = fast_exp2(m - (m_new == kNegInf ? 0.f : m_new));  // 0 while the row has seen no key
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
        m = m_new;
        off = m_new == kNegInf ? 0.f : m_new;
        threshold = (m_new + kFastRange) * inv_scale_log2;
      }
    }
#pragma unroll
    for (int hf = 0; hf < N / 32; ++hf) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = sc[2 * hf + (i >> 2)][i & 3];
        p[i] = fast_exp2(MODE == 0 ? fmaf(x, scale_log2, -off) : x - off);
      }
      if constexpr (MODE == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          l[i & 3] += p[i];
          p[i] = p[i] == 0.f ? 0.f : p[i] * vs[2 * hf + (i >> 2)][i & 3];  // a hidden key's scale may be anything
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
        hi[hf][i >> 1] = __builtin_amdgcn_perm(cut[1], cut[0], 0x07060302u);
        lo[hf][i >> 1] = pack_bf16x2(rest[0], rest[1]);
      }
      if constexpr (MODE == 0) {  // the sums on the matrix cores, of the values that the product uses
        l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, hi[hf]), l, 0, 0, 0);
        l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, lo[hf]), l, 0, 0, 0);
      }
    }
  }

  // O^T += V^T . P^T over N keys whose V stands row-major in LDS.
  template <int N>
  __device__ __forceinline__ void product(const uint16_t* sv, int tr_off, int pitch, const u32x4 (&hi)[N / 32],
                                          const u32x4 (&lo)[N / 32]) {
#pragma unroll
    for (int hf = 0; hf < N / 32; ++hf)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 vop = read_v_operand<bf16x8>(sv + 32 * pitch * hf, tr_off, pitch, 16 * dt);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, __builtin_bit_cast(bf16x8, hi[hf]), acc[dt], 0, 0, 0);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, __builtin_bit_cast(bf16x8, lo[hf]), acc[dt], 0, 0, 0);
      }
  }

  __device__ __forceinline__ float sum(int mode) const {
    return mode == 0 ? l[0] : sum_over_rows_swap(l[0] + l[1] + l[2] + l[3]);
  }
};

template <int D>
__device__ __forceinline__ bf16x8 bf16_ones() {
  bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
  if constexpr (D == 64) asm volatile("" : "+v"(ones));  // kept in registers, where there is room
  return ones;
}

template <int D>
struct PrefixSmem {
  static constexpr int KT = kPrefixStage, P = D + 16;  // keys of a stage, elements between its rows
  static constexpr int kTiles = 2 * 2 * KT * P * 2;  // [buffer][K, V][key][P]
  static constexpr int kOwnPitch = D + 8;
  static constexpr int kOwnTiles = kPrefixWaves * 32 * kOwnPitch * 2;  // [wave][key][P] of V
  static constexpr int kBytes = kTiles > kOwnTiles ? kTiles : kOwnTiles;
};

// A prefix item: 8 / KW waves side by side over 16 rows each, KW one after the other over a stage's keys.
template <int D, int MODE, int KW, int NPRE>
__device__ __forceinline__ void prefix_item(const PrefixArgs& a, char* smem, float (*sscale)[2][kPrefixStage], int* bids, int index) {
  const float scale_log2 = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, a.scale_log2)));
  const bool k_f32 = a.ks_f32, v_f32 = a.vs_f32;
  constexpr int KT = kPrefixStage, KPW = KT / KW, P = D + 16, KS = D / 32, DT = D / 16;
  constexpr int PT = kPrefixThreads, RW = kPrefixWaves / KW, ROWS = 16 * RW;
  constexpr int CH = MODE == 0 ? 8 : 16, CPK = D / CH, NCH = KT * CPK;  // 16-byte parts of a key, of a stage
  constexpr int LPT = (NCH + PT - 1) / PT;
  uint16_t(*sm)[2][KT * P] = (uint16_t(*)[2][KT * P]) smem;
  const int item = index, tid = threadIdx.x, lane = tid & 63, r = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave / RW, rw = wave % RW;
  const int4 i0 = *(const int4*)(a.items + 8 * (int64_t)item), i1 = *(const int4*)(a.items + 8 * (int64_t)item + 4);
  const int table_row = min(max(i0.x, 0), a.S - 1), first_member = max(i0.y, 0), M = max(i0.z, 1), m0 = max(i0.w, 0);
  const int h = min(max(i1.x, 0), a.Hkv - 1), k_lo = max(i1.y, 0), k_hi = min(min(i1.z, a.max_ctx), k_lo + kPrefixMaxChunk);
  const int nkeys = k_hi - k_lo, G = a.G;
  if (nkeys <= 0) return;  // (never in a list of sipa_prefix_plan)

  const int32_t* table = a.bt + (int64_t)table_row * a.bt_ss;
  const int first_col = k_lo >> a.log_b;
  for (int i = tid; i << a.log_b < nkeys; i += PT) bids[i] = min(max(table[min(first_col + i, a.bt_w - 1)], 0), a.nb - 1);
  const int m = m0 + 16 * rw + r, at = min(m, M - 1);
  const bool valid = m0 + 16 * rw < M;  // wave-uniform: some row of the tile is there
  bf16x8 qop[KS];
  {
    const int i = at / G, s = min(max(a.members[min(first_member + i, a.num_members - 1)], 0), a.S - 1);
#pragma unroll
    for (int j = 0; j < KS; ++j)
      qop[j] = __builtin_bit_cast(
          bf16x8, *(const u32x4*)(a.q + (int64_t)s * a.q_ss + (int64_t)(h * G + at - i * G) * a.q_sh + 32 * j + 8 * q4));
  }
  const float inv_scale_log2 = MODE == 0 ? 1.f / scale_log2 : 1.f;
  RowState<D> st;
  st.clear();
  const int tr_off = tr16_offset(r, q4, P);
  const bf16x8 ones = bf16_ones<D>();
  __syncthreads();  // block ids

  const int ntiles = (nkeys + KT - 1) / KT;
  u32x4 rk[NPRE][LPT], rv[NPRE][LPT];
  u32x2 rs[NPRE];
  // A thread's parts of a stage keep their place in their blocks from stage to stage (a stage is whole blocks): what changes
  // is the block id. Keys past the item's end are read too, inside its last block; they are hidden, and their V is zero.
  const int es = MODE == 0 ? 2 : 1, last_id = (nkeys - 1) >> a.log_b;
  const uint32_t kv_bytes = (uint32_t)a.kv_sn * es;  // of a block (host-checked)
  const uint8_t* kbase[LPT];
  const int64_t v_from_k = (const uint8_t*)a.v - (const uint8_t*)a.k;
  int part_id[LPT];
#pragma unroll
  for (int i = 0; i < LPT; ++i) {
    const int c = tid + PT * i, key = c / CPK;
    const int64_t e = ((int64_t)h * a.kv_sh + (key & ((1 << a.log_b) - 1)) * D + CH * (c % CPK)) * es;
    kbase[i] = (const uint8_t*)a.k + e;
    part_id[i] = key >> a.log_b;
  }
  // Threads 0 .. KT - 1 bring a stage's scales of K, the next KT those of V. (Chosen among copies: a choice among the arguments'
  // addresses puts them into memory, whose own address comes from the launch's packet on the host, at 50 ns a workgroup: 64
  // sequences of 500 tokens 18.9 -> 10.6 us.)
  const void *k_scales = a.ks, *v_scales = a.vs;
  const int64_t ks_head = (int64_t)h * a.ks_sh, vs_head = (int64_t)h * a.vs_sh, ks_sn = a.ks_sn, vs_sn = a.vs_sn;
  const bool of_k = tid < KT, scale_f32 = of_k ? k_f32 : v_f32;
  const void* scales = (const char*)(of_k ? k_scales : v_scales) +
                       ((of_k ? ks_head : vs_head) + (tid & ((1 << a.log_b) - 1))) * (scale_f32 ? 4 : 2);
  const int64_t scale_block = of_k ? ks_sn : vs_sn;
  auto gload = [&](int set, int t) {
#pragma unroll
    for (int i = 0; i < LPT; ++i) {
      if (NCH % PT != 0 && tid + PT * i >= NCH) break;
      const uint64_t b = (uint64_t)(uint32_t)bids[min((KT * t >> a.log_b) + part_id[i], last_id)] * kv_bytes;
      rk[set][i] = *(const u32x4*)(kbase[i] + b);
      rv[set][i] = *(const u32x4*)(kbase[i] + b + v_from_k);
    }
    if constexpr (MODE == 1) {
      if (tid < 2 * KT)
        rs[set] = load_scale(scales, scale_f32, bids[min((KT * t >> a.log_b) + (tid % KT >> a.log_b), last_id)] * scale_block);
    }
  };
  auto sstore = [&](int set, int t) {
    const int buf = t & 1;
#pragma unroll
    for (int i = 0; i < LPT; ++i) {
      const int c = tid + PT * i;
      if (NCH % PT != 0 && c >= NCH) break;
      const int key = c / CPK, e = key * P + CH * (c % CPK);
      const u32x4 k = rk[set][i];
      u32x4 v = rv[set][i];
      if (KT * t + key >= nkeys) v = u32x4{0, 0, 0, 0};
      if constexpr (MODE == 0) {
        *(u32x4*)(&sm[buf][0][e]) = k;
        *(u32x4*)(&sm[buf][1][e]) = v;
      } else {
        // Odd lanes store their second half first at head_dim 64, as 16 bytes of each 32 use half the banks. The halves change
        // places by their differing bits.
        const int odd = D == 64 ? tid & 1 : 0;
        const uint32_t swap = -(uint32_t)odd;
        auto store = [&](uint16_t* to, u32x4 x) {
          const uint32_t d0 = (x[0] ^ x[2]) & swap, d1 = (x[1] ^ x[3]) & swap;
          *(u32x4*)(to + 8 * odd) = tree_codes(x[0] ^ d0, x[1] ^ d1);
          *(u32x4*)(to + 8 - 8 * odd) = tree_codes(x[2] ^ d0, x[3] ^ d1);
        };
        store(&sm[buf][0][e], k);
        store(&sm[buf][1][e], v);
      }
    }
    if constexpr (MODE == 1) {
      if (tid < 2 * KT) sscale[buf][tid / KT][tid % KT] = one_scale(rs[set], scale_f32) * (of_k ? scale_log2 : 1.f);
    }
  };
  // At head_dim 128 half of the wave's keys at a time: the scores of 64 would not fit the registers of two workgroups a CU.
  constexpr int SUB = D == 64 ? KPW : 32, SMT = SUB / 16;
  auto tile = [&](int t) {
    const int buf = t & 1;
#pragma unroll
    for (int part = 0; part < KPW / SUB; ++part) {
      const int first = KPW * kw + SUB * part, x0 = KT * t + first;  // the keys' place in the stage, in the item
      if (x0 >= nkeys || !valid) return;  // wave-uniform
      const uint16_t* sk = sm[buf][0] + first * P;
      const uint16_t* sv = sm[buf][1] + first * P;
      f32x4 sc[SMT], vs[SMT];  // row (mt, q4, i) holds key 16 mt + 4 q4 + i
#pragma unroll
      for (int mt = 0; mt < SMT; ++mt) {
        sc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const bf16x8 kop = *(const bf16x8*)(sk + (16 * mt + r) * P + 32 * j + 8 * q4);
          sc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop, qop[j], sc[mt], 0, 0, 0);
        }
        if constexpr (MODE == 1) {
          sc[mt] *= *(const f32x4*)(sscale[buf][0] + first + 16 * mt + 4 * q4);  // log2 units
          vs[mt] = *(const f32x4*)(sscale[buf][1] + first + 16 * mt + 4 * q4);
        }
      }
      if (x0 + SUB > nkeys) {
#pragma unroll
        for (int mt = 0; mt < SMT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (x0 + 16 * mt + 4 * q4 + i >= nkeys) sc[mt][i] = kNegInf;
      }
      u32x4 hi[SUB / 32], lo[SUB / 32];
      st.template add<MODE, SUB>(sc, scale_log2, inv_scale_log2, ones, vs, hi, lo);
      st.template product<SUB>(sv, tr_off, P, hi, lo);
    }
  };
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
  float l = st.sum(MODE);
  if (l != l) st.m = 0.f;  // NaN scores never raise the max: the merges see the row by its sum
  if constexpr (KW > 1) {
    // The key waves' states join in LDS (the tile buffers are free after the last barrier).
    constexpr int XS = DT * 4 + 4;  // floats of a lane: O, m, l
    static_assert((KW - 1) * RW * 64 * XS * 4 <= PrefixSmem<D>::kTiles, "the states fit the tile buffers");
    float* xs = (float*)smem;
    if (kw > 0) {
      float* x = xs + (((kw - 1) * RW + rw) * 64 + lane) * XS;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *(f32x4*)(x + 4 * dt) = st.acc[dt];
      x[4 * DT] = st.m;
      x[4 * DT + 1] = l;
    }
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int k = 1; k < KW; ++k) {
        const float* x = xs + (((k - 1) * RW + rw) * 64 + lane) * XS;
        const float m1 = x[4 * DT], l1 = x[4 * DT + 1], top = vmax(st.m, m1);
        if (top == kNegInf) continue;
        const float f0 = fast_exp2(st.m - top), f1 = fast_exp2(m1 - top);
        l = f0 * l + f1 * l1;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) st.acc[dt] = f0 * st.acc[dt] + f1 * *(const f32x4*)(x + 4 * dt);
        st.m = top;
      }
    }
  }
  if (kw > 0 || m >= M) return;
  const int64_t slot = (int64_t)min(max(i1.w, 0), a.num_items - 1) * ROWS + 16 * rw + r;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *(GlobalF32x4*)(a.st_o + slot * D + 16 * dt + 4 * q4) = st.acc[dt];
  if (q4 == 0) *(GlobalU64*)(a.st_ml + slot) = __builtin_bit_cast(uint64_t, float2{st.m, l});
}

// An own piece, a wave: 32 keys at a time in two halves, K straight into the operand's registers, V through LDS of the wave's own.
// Registers hold NH halves: a half's are loaded again for a later one as soon as its K is in the scores and its V in LDS.
template <int D, int MODE, int NH>
__device__ __forceinline__ void own_piece(const PrefixArgs& a, char* smem, int index) {
  const float scale_log2 = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, a.scale_log2)));
  const bool k_f32 = a.ks_f32, v_f32 = a.vs_f32;
  constexpr int KS = D / 32, DT = D / 16, P = D + 8;
  constexpr int VCH = MODE == 0 ? 8 : 16, VPK = D / VCH, VL = (16 * VPK + 63) / 64;  // 16-byte parts of V: a key's, a lane's of a half
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int piece = __builtin_amdgcn_readfirstlane(index * kPrefixWaves + wave);
  if (piece >= a.num_pieces) return;
  const int4 i0 = *(const int4*)(a.pieces + 8 * (int64_t)piece), i1 = *(const int4*)(a.pieces + 8 * (int64_t)piece + 4);
  const int s = min(max(__builtin_amdgcn_readfirstlane(i0.x), 0), a.S - 1), h = min(max(__builtin_amdgcn_readfirstlane(i0.y), 0), a.Hkv - 1);
  const int sp = max(__builtin_amdgcn_readfirstlane(i0.z), 0), planned = max(__builtin_amdgcn_readfirstlane(i0.w), 1);
  const int tokens = max(__builtin_amdgcn_readfirstlane(i1.x), 0), G = a.G;
  bf16x8 qop[KS];
#pragma unroll
  for (int j = 0; j < KS; ++j)
    qop[j] = __builtin_bit_cast(bf16x8, *(const u32x4*)(a.q + (int64_t)s * a.q_ss + (int64_t)(h * G + min(r, G - 1)) * a.q_sh +
                                                        32 * j + 8 * q4));
  const OwnKeys own = own_keys(a, s, tokens, planned);
  if (sp >= own.pieces) return;
  const int lo_key = own.shared + sp * own.chunk, end = min(lo_key + own.chunk, own.ctx);
  const int32_t* table = a.bt + (int64_t)s * a.bt_ss;
  const int last_col = min((end - 1) >> a.log_b, a.bt_w - 1);
  const float inv_scale_log2 = MODE == 0 ? 1.f / scale_log2 : 1.f;
  RowState<D> st;
  st.clear();
  uint16_t* sv = (uint16_t*)smem + wave * 32 * P;
  const int tr_off = tr16_offset(r, q4, P);
  const bf16x8 ones = bf16_ones<D>();
  const int halves = 2 * ((end - lo_key + 31) / 32);
  u32x4 rk[NH][KS], rv[NH][VL];
  u32x4 rks[NH], rvs[NH];
  // the id of the block that half i, 16 keys, is inside; halves past the end read the last block again
  auto id_of = [&](int i) { return table[min((lo_key + 16 * i) >> a.log_b, last_col)]; };
  const int k_off = r * D + 8 * q4;
  auto load = [&](int set, int i, int entry) {
    const int id = __builtin_amdgcn_readfirstlane(min(max(entry, 0), a.nb - 1));
    const int off = (lo_key + 16 * i) & ((1 << a.log_b) - 1);
    const int64_t base = (int64_t)h * a.kv_sh + (int64_t)id * a.kv_sn + off * D;
    const uint8_t* k = (const uint8_t*)a.k + base * (MODE == 0 ? 2 : 1);
    const uint8_t* v = (const uint8_t*)a.v + base * (MODE == 0 ? 2 : 1);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      if constexpr (MODE == 0) {
        rk[set][j] = *(const u32x4*)(k + 2 * (k_off + 32 * j));
      } else {
        const u32x2 c = *(const u32x2*)(k + k_off + 32 * j);
        rk[set][j] = u32x4{c[0], c[1], 0, 0};
      }
    }
#pragma unroll
    for (int x = 0; x < VL; ++x)
      if (16 * VPK % 64 == 0 || lane + 64 * x < 16 * VPK) rv[set][x] = *(const u32x4*)(v + 16 * (lane + 64 * x));
    if constexpr (MODE == 1) {
      rks[set] = load_scales(a.ks, k_f32, (int64_t)h * a.ks_sh + (int64_t)id * a.ks_sn + off + 4 * q4);
      rvs[set] = load_scales(a.vs, v_f32, (int64_t)h * a.vs_sh + (int64_t)id * a.vs_sn + off + 4 * q4);
    }
  };
  // Table entries are loaded a half ahead of the keys they are for, and before those of the half between: a wait for one is then
  // no wait for keys that are still to come.
  int first[NH + 1];
#pragma unroll
  for (int i = 0; i <= NH; ++i) first[i] = id_of(i);
#pragma unroll
  for (int i = 0; i < NH; ++i) load(i, i, first[i]);
  int id = first[NH];
  for (int i0 = 0; i0 < halves; i0 += 2) {
    f32x4 sc[2], vs[2];
    wave_sync();  // the last tile's reads of V
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int set = half % NH, i = i0 + half, x0 = lo_key + 16 * i;
#pragma unroll
      for (int x = 0; x < VL; ++x) {
        const int c = lane + 64 * x, key = c / VPK;
        if (16 * VPK % 64 != 0 && c >= 16 * VPK) break;
        u32x4 v = rv[set][x];
        if (x0 + key >= end) v = u32x4{0, 0, 0, 0};
        uint16_t* to = sv + (16 * half + key) * P + VCH * (c % VPK);
        if constexpr (MODE == 0) {
          *(u32x4*)to = v;
        } else {
          *(u32x4*)to = tree_codes(v[0], v[1]);
          *(u32x4*)(to + 8) = tree_codes(v[2], v[3]);
        }
      }
      sc[half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const u32x4 k = MODE == 0 ? rk[set][j] : tree_codes(rk[set][j][0], rk[set][j][1]);
        sc[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), qop[j], sc[half], 0, 0, 0);
      }
      if constexpr (MODE == 1) {
        sc[half] *= four_scales(rks[set], k_f32) * scale_log2;
        vs[half] = four_scales(rvs[set], v_f32);
        asm volatile("" : "+v"(vs[half]));  // now: the registers are loaded again below
      }
      if (x0 + 16 > end) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (x0 + 4 * q4 + x >= end) sc[half][x] = kNegInf;
      }
      const int next = id_of(i + NH + 1);
      load(set, i + NH, id);
      id = next;
    }
    u32x4 hi[1], lo[1];
    st.template add<MODE, 32>(sc, scale_log2, inv_scale_log2, ones, vs, hi, lo);
    wave_sync();  // V has been stored
    st.template product<32>(sv, tr_off, P, hi, lo);
  }
  float l = st.sum(MODE);
  if (l != l) st.m = 0.f;  // NaN scores never raise the max: the merge sees the row by its sum
  if (r >= G) return;
  const int64_t slot = (int64_t)a.num_items * a.tile_rows + (int64_t)min(max(__builtin_amdgcn_readfirstlane(i1.y), 0), a.num_pieces - 1) * G + r;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *(GlobalF32x4*)(a.st_o + slot * D + 16 * dt + 4 * q4) = st.acc[dt];
  if (q4 == 0) *(GlobalU64*)(a.st_ml + slot) = __builtin_bit_cast(uint64_t, float2{st.m, l});
}

template <int D, int MODE, int KW, int NPRE>
__global__ void __launch_bounds__(kPrefixThreads, 4) prefix_attention_kernel(const PrefixArgs a) {
  __shared__ __align__(16) char smem[PrefixSmem<D>::kBytes];
  __shared__ __align__(16) float sscale[MODE == 0 ? 1 : 2][2][kPrefixStage];
  __shared__ int bids[kPrefixMaxChunk / 16];
  if ((int)blockIdx.x < a.num_items) prefix_item<D, MODE, KW, NPRE>(a, smem, sscale, bids, blockIdx.x);
  else own_piece<D, MODE, D == 64 ? 2 : 1>(a, smem, (int)blockIdx.x - a.num_items);
}

// Joins the parts of a row, a wave: lane (part, 4 channels), 256 / D parts side by side. A row without any key gets zeros.
template <int D>
__global__ void __launch_bounds__(256) prefix_merge_kernel(const PrefixArgs a) {
  constexpr int Q = D / 4, ROWS = 64 / Q, U = 8;  // parts side by side, of which a lane takes U at a time
  const int lane = threadIdx.x & 63, row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), Hq = a.Hkv * a.G;
  if (row >= a.S * Hq) return;
  const int s = row / Hq, hq = row - s * Hq, h = hq / a.G, g = hq - h * a.G, c = lane % Q, side = lane / Q;
  const int4 i0 = *(const int4*)(a.rows + 8 * (int64_t)s), i1 = *(const int4*)(a.rows + 8 * (int64_t)s + 4);
  const OwnKeys own = own_keys(a, s, i0.x, max(i1.z, 1));
  const int np = own.shared > 0 ? i0.w : 0, m = i0.y + g, tile = m / a.tile_rows, n = np + own.pieces;
  const int64_t p0 = ((int64_t)i0.z + (int64_t)(h * i1.x + tile) * np) * a.tile_rows + (m - tile * a.tile_rows);
  const int64_t s0 = (int64_t)a.num_items * a.tile_rows + ((int64_t)i1.y + (int64_t)h * i1.z) * a.G + g;
  float M = kNegInf, L = 0.f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = side; j0 < n; j0 += ROWS * U) {
    float ms[U], ls[U];
    f32x4 os[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(j0 + ROWS * u, n - 1);
      const int64_t i = j < np ? p0 + (int64_t)j * a.tile_rows : s0 + (int64_t)(j - np) * a.G;
      const float2 ml = a.st_ml[i];
      ms[u] = ml.x, ls[u] = ml.y;
      os[u] = *(const f32x4*)(a.st_o + i * D + 4 * c);
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, j0 + ROWS * u < n ? ms[u] : kNegInf);
    if (top == kNegInf) continue;
    const float f = fast_exp2(M - top);
    L *= f;
    O *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j0 + ROWS * u >= n || ms[u] == kNegInf) continue;  // a part without a key for the row
      const float e = fast_exp2(ms[u] - top);
      L += e * ls[u];
      O += e * os[u];
    }
    M = top;
  }
  auto join = [&](int o) {
    const float m1 = __shfl_xor(M, o), l1 = __shfl_xor(L, o), top = fmaxf(M, m1);
    f32x4 o1;
#pragma unroll
    for (int i = 0; i < 4; ++i) o1[i] = __shfl_xor(O[i], o);
    // (an empty side's O is 0, but its factor would be NaN)
    const float f0 = M == kNegInf ? 0.f : fast_exp2(M - top), f1 = m1 == kNegInf ? 0.f : fast_exp2(m1 - top);
    L = f0 * L + f1 * l1;
    O = f0 * O + f1 * o1;
    M = top;
  };
#pragma unroll
  for (int o = Q; o < 64; o *= 2) join(o);
  if (side > 0) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *(u32x2*)(a.out + (int64_t)s * a.o_ss + (int64_t)hq * a.o_sh + 4 * c) =
      u32x2{pack_bf16x2(O[0] * inv, O[1] * inv), pack_bf16x2(O[2] * inv, O[3] * inv)};
}

}  // namespace sipa

using namespace sipa;

static int prefix_check(const sipa_prefix_params* p) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_prefix_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_prefix_params (%d bytes)", (int)sizeof(sipa_prefix_params));
  SIPA_CHECK(p->num_seqs >= 0 && p->num_kv_heads > 0 && p->num_q_heads > 0 && p->num_q_heads % p->num_kv_heads == 0, SIPA_EINVAL,
             "bad sequence or head counts");
  SIPA_CHECK(p->num_q_heads / p->num_kv_heads <= kMaxGroup, SIPA_EUNSUPPORTED, "GQA group %d > %d",
             p->num_q_heads / p->num_kv_heads, kMaxGroup);
  SIPA_CHECK(p->head_dim == 64 || p->head_dim == 128, SIPA_EUNSUPPORTED, "head_dim %d not in {64, 128}", p->head_dim);
  SIPA_CHECK(p->block_size == 16 || p->block_size == 32 || p->block_size == 64, SIPA_EUNSUPPORTED,
             "block_size %d not in {16, 32, 64}", p->block_size);
  SIPA_CHECK(p->max_context > 0 && p->max_context <= 1 << 24, SIPA_EUNSUPPORTED, "max_context %d outside [1, 2^24]", p->max_context);
  SIPA_CHECK(p->kv_mode == SIPA_KV_PLAIN || p->kv_mode == SIPA_KV_INT8_TOKEN, SIPA_EUNSUPPORTED, "kv_mode %d", p->kv_mode);
  SIPA_CHECK((int64_t)p->num_seqs * p->num_q_heads * p->head_dim <= 0x3fffffff, SIPA_EUNSUPPORTED, "%d sequences of %d heads",
             p->num_seqs, p->num_q_heads);
  return SIPA_OK;
}

struct PrefixStates {
  int64_t ml, total;  // byte offsets into the workspace
};

static PrefixStates prefix_workspace(const sipa_prefix_params* p, const sipa_prefix_layout& l) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  const int64_t n = (int64_t)l.num_items * l.tile_rows + (int64_t)l.num_pieces * (p->num_q_heads / p->num_kv_heads);
  const int64_t ml = up(n * p->head_dim * 4);
  return PrefixStates{ml, ml + up(n * 8)};
}

extern "C" int32_t sipa_prefix_plan(const sipa_prefix_params* p, int32_t num_groups, const int32_t* group_starts,
                                    const int32_t* members, const int32_t* tokens, const int32_t* context_lens,
                                    int32_t* plan, int64_t capacity, sipa_prefix_layout* layout) {
  int rc = prefix_check(p);
  if (rc != SIPA_OK) return rc;
  SIPA_CHECK(layout != nullptr && num_groups >= 0 && (num_groups == 0 || (group_starts && members && tokens)), SIPA_EINVAL,
             "NULL pointer or negative group count");
  const int S = p->num_seqs, G = p->num_q_heads / p->num_kv_heads, H = p->num_kv_heads;
  SIPA_CHECK(num_groups == 0 || group_starts[0] == 0, SIPA_EINVAL, "group_starts begin at %d", num_groups ? group_starts[0] : 0);
  const int num_members = num_groups ? group_starts[num_groups] : 0;
  // groups that share anything: two members at least, one block
  auto count_of = [&](int g) { return group_starts[g + 1] - group_starts[g]; };
  auto shares = [&](int g) { return count_of(g) >= 2 && tokens[g] > 0; };
  auto length = [&](int s) { return context_lens == nullptr ? p->max_context : std::min(std::max(context_lens[s], 0), p->max_context); };
  int64_t most_rows = 0, own = 0;  // own: keys that are read for one sequence
  for (int s = 0; s < S; ++s) own += length(s);
  for (int g = 0; g < num_groups; ++g) {
    SIPA_CHECK(count_of(g) >= 0 && group_starts[g + 1] <= S, SIPA_EINVAL, "group %d has rows %d .. %d of %d", g, group_starts[g],
               group_starts[g + 1], S);
    SIPA_CHECK(tokens[g] >= 0 && tokens[g] <= p->max_context && tokens[g] % p->block_size == 0, SIPA_EINVAL,
               "group %d shares %d tokens: whole blocks of %d within max_context %d", g, tokens[g], p->block_size, p->max_context);
    for (int i = group_starts[g]; i < group_starts[g + 1]; ++i) {
      SIPA_CHECK(members[i] >= 0 && members[i] < S, SIPA_EINVAL, "group %d has row %d of %d", g, members[i], S);
      if (shares(g) && length(members[i]) >= tokens[g]) own -= tokens[g];
    }
    if (shares(g)) most_rows = std::max<int64_t>(most_rows, (int64_t)count_of(g) * G);
  }
  const int found = sipa_device_cu_count(-1), cus = found > 0 ? found : 256;  // planned without a GPU: an MI355X's
  sipa_prefix_layout l = {};
  l.tile_rows = most_rows <= 64 ? 64 : 128;
  const int kt = kPrefixStage;
  auto tiles_of = [&](int g) { return ((int64_t)count_of(g) * G + l.tile_rows - 1) / l.tile_rows; };
  int64_t work = 0;  // keys times row tiles
  for (int g = 0; g < num_groups; ++g)
    if (shares(g)) work += (int64_t)H * tiles_of(g) * tokens[g];
  // Two workgroups a CU are resident: the own pieces take as many as they need with 64 keys a piece, or 128 .. 512 where those
  // would not all be resident, and the items share the rest, half of a CU's at least, with 128 keys each at least. (64 beams of
  // 4096 + 300 tokens: 512 items beside 75 workgroups of pieces 19.0 us, 352 14.5; two documents of 30016 tokens, 37 sequences
  // each: 256 items 45.8, 480 33. Pieces of 64 / 128 keys: 128 sequences of 100 tokens 17.2 / 21.1, 200 of 1000 44 / 40.)
  int64_t piece = 64;
  while (piece < 512 && own * H > piece * 8 * 2 * cus) piece *= 2;
  const int64_t free = std::max<int64_t>(2 * cus - (own * H / piece + S * H) / 8, cus / 2);
  const int64_t share = std::max<int64_t>(128, (work + free - 1) / free);
  struct Cut {
    int64_t n, chunk;
  };
  auto cut_of = [&](int g) {
    const int64_t n = std::max<int64_t>((tokens[g] + share - 1) / share, (tokens[g] + kPrefixMaxChunk - 1) / kPrefixMaxChunk);
    const int64_t chunk = ((tokens[g] + n - 1) / n + kt - 1) / kt * kt;
    return Cut{(tokens[g] + chunk - 1) / chunk, chunk};
  };
  int64_t items = 0;
  for (int g = 0; g < num_groups; ++g)
    if (shares(g)) items += H * tiles_of(g) * cut_of(g).n;
  auto pieces_of = [&](int s, int shared) {  // for a KV head; one at least, for lengths that come to be another
    const int n = length(s) >= shared ? length(s) - shared : length(s);
    return std::max<int64_t>(1, (n + piece - 1) / piece);
  };
  // The rows, in the plan's place or counted alone.
  int64_t pieces = 0;
  for (int s = 0; s < S; ++s) pieces += H * pieces_of(s, 0);
  for (int g = 0; g < num_groups; ++g)
    if (shares(g))
      for (int i = group_starts[g]; i < group_starts[g + 1]; ++i) pieces += H * (pieces_of(members[i], tokens[g]) - pieces_of(members[i], 0));
  SIPA_CHECK(pieces >= 0 && items + pieces <= 0x7fffffff / 128, SIPA_EUNSUPPORTED, "%lld items exceed the grid limit",
             (long long)(items + pieces));
  l.num_items = (int)items;
  l.num_pieces = (int)pieces;
  l.num_members = num_members;
  l.plan_ints = 8 * (items + pieces + S) + num_members;
  l.workspace_bytes = prefix_workspace(p, l).total;
  *layout = l;
  if (plan == nullptr) return SIPA_OK;
  SIPA_CHECK(capacity >= l.plan_ints, SIPA_EINVAL, "the plan takes %lld values, room for %lld", (long long)l.plan_ints,
             (long long)capacity);
  int32_t* pcs = plan + 8 * items;
  int32_t* rows = pcs + 8 * pieces;
  for (int64_t i = 0; i < 8 * (int64_t)S; ++i) rows[i] = i % 8 == 7 ? -1 : 0;
  int64_t at = 0;
  for (int g = 0; g < num_groups; ++g) {
    const int a0 = group_starts[g], count = count_of(g);
    for (int i = 0; i < count; ++i) {
      int32_t* r = rows + 8 * (int64_t)members[a0 + i];
      SIPA_CHECK(r[7] < 0, SIPA_EINVAL, "row %d in two groups, or twice in one", members[a0 + i]);
      r[7] = g;
    }
    if (!shares(g)) continue;
    const int64_t tiles = tiles_of(g);
    const Cut cut = cut_of(g);
    for (int i = 0; i < count; ++i) {
      int32_t* r = rows + 8 * (int64_t)members[a0 + i];
      r[0] = tokens[g], r[1] = i * G, r[2] = (int)at, r[3] = (int)cut.n, r[4] = (int)tiles;
    }
    // State (h, tile, split). Workgroup L is dealt to XCD L % 8: the row tiles of the same keys come eight apart.
    const int64_t units = H * cut.n;
    for (int64_t u0 = 0, put = at; u0 < units; u0 += 8)
      for (int64_t t = 0; t < tiles; ++t)
        for (int64_t u = u0; u < std::min<int64_t>(u0 + 8, units); ++u) {
          const int64_t h = u / cut.n, x = u - h * cut.n;
          int32_t* it = plan + 8 * put++;
          it[0] = members[a0], it[1] = a0, it[2] = count * G, it[3] = (int)(t * l.tile_rows);
          it[4] = (int)h, it[5] = (int)(x * cut.chunk), it[6] = (int)std::min<int64_t>((x + 1) * cut.chunk, tokens[g]);
          it[7] = (int)(at + (h * tiles + t) * cut.n + x);
        }
    at += units * tiles;
  }
  int64_t put = 0;
  for (int s = 0; s < S; ++s) {
    int32_t* r = rows + 8 * (int64_t)s;
    const int64_t n = pieces_of(s, r[0]);
    r[5] = (int)put, r[6] = (int)n;
    for (int h = 0; h < H; ++h)
      for (int64_t x = 0; x < n; ++x, ++put) {
        int32_t* q = pcs + 8 * put;
        q[0] = s, q[1] = h, q[2] = (int)x, q[3] = (int)n, q[4] = r[0], q[5] = (int)put, q[6] = q[7] = 0;
      }
  }
  for (int i = 0; i < num_members; ++i) rows[8 * (int64_t)S + i] = members[i];
  return SIPA_OK;
}

template <int D, int MODE>
static void launch_prefix(int tile_rows, dim3 grid, hipStream_t st, const PrefixArgs& a) {
  constexpr int NPRE = D == 64 ? 3 : 2;
  if (tile_rows == 64) hipLaunchKernelGGL((prefix_attention_kernel<D, MODE, 2, NPRE>), grid, dim3(kPrefixThreads), 0, st, a);
  else hipLaunchKernelGGL((prefix_attention_kernel<D, MODE, 1, NPRE>), grid, dim3(kPrefixThreads), 0, st, a);
  hipLaunchKernelGGL((prefix_merge_kernel<D>), dim3((unsigned)((a.S * a.Hkv * a.G + 3) / 4)), dim3(256), 0, st, a);
}

extern "C" int32_t sipa_prefix_attention(const sipa_prefix_params* p, void* stream) {
  int rc = prefix_check(p);
  if (rc != SIPA_OK) return rc;
  if (p->num_seqs == 0) return SIPA_OK;
  SIPA_CHECK(p->scale > 0.f && p->scale < __builtin_inff(), SIPA_EINVAL,
             "scale %g must be positive and finite (the kernel takes maxima of the unscaled scores)", (double)p->scale);
  SIPA_CHECK(p->bt_width > 0 && (int64_t)p->bt_width * p->block_size >= p->max_context, SIPA_EINVAL,
             "block_tables rows of %d entries cannot cover max_context %d", p->bt_width, p->max_context);
  SIPA_CHECK(p->q && p->k_cache && p->v_cache && p->block_tables && p->context_lens && p->out && p->plan && p->num_blocks > 0,
             SIPA_EINVAL, "NULL pointer or empty pool");
  SIPA_CHECK(((uintptr_t)p->q & 15) == 0 && p->q_stride_s % 8 == 0 && p->q_stride_h % 8 == 0, SIPA_EINVAL,
             "q rows must be 16-byte aligned");
  SIPA_CHECK(((uintptr_t)p->out & 7) == 0 && p->out_stride_s % 4 == 0 && p->out_stride_h % 4 == 0, SIPA_EINVAL,
             "out rows must be 8-byte aligned");
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
  const sipa_prefix_layout& l = p->layout;
  SIPA_CHECK((l.tile_rows == 64 || l.tile_rows == 128) && l.num_items >= 0 && l.num_members >= 0 &&
                 l.num_pieces >= (int64_t)p->num_seqs * p->num_kv_heads && (int64_t)l.num_items + l.num_pieces <= 0x7fffffff / 128 &&
                 ((uintptr_t)p->plan & 15) == 0, SIPA_EINVAL, "the layout is not one of sipa_prefix_plan for these sizes");
  const PrefixStates w = prefix_workspace(p, l);
  SIPA_CHECK(p->workspace != nullptr && ((uintptr_t)p->workspace & 255) == 0 && p->workspace_bytes >= w.total, SIPA_EWORKSPACE,
             "a 256-byte aligned workspace of %lld bytes is needed (have %lld)", (long long)w.total, (long long)p->workspace_bytes);
  PrefixArgs a;
  a.q = (const uint16_t*)p->q;
  a.q_ss = p->q_stride_s;
  a.q_sh = p->q_stride_h;
  a.k = p->k_cache;
  a.v = p->v_cache;
  a.kv_sh = p->kv_stride_h;
  a.kv_sn = p->kv_stride_n;
  a.bt = p->block_tables;
  a.bt_ss = p->bt_stride_s;
  a.bt_w = p->bt_width;
  a.ctx = p->context_lens;
  a.out = (uint16_t*)p->out;
  a.o_ss = p->out_stride_s;
  a.o_sh = p->out_stride_h;
  a.ks = p->k_scale;
  a.vs = p->v_scale;
  a.ks_f32 = p->k_scale_dtype == SIPA_F32;
  a.vs_f32 = p->v_scale_dtype == SIPA_F32;
  a.ks_sh = p->ks_stride_h;
  a.ks_sn = p->ks_stride_n;
  a.vs_sh = p->vs_stride_h;
  a.vs_sn = p->vs_stride_n;
  a.items = p->plan;
  a.pieces = p->plan + 8 * (int64_t)l.num_items;
  a.rows = a.pieces + 8 * (int64_t)l.num_pieces;
  a.members = a.rows + 8 * (int64_t)p->num_seqs;
  a.num_items = l.num_items;
  a.num_pieces = l.num_pieces;
  a.num_members = l.num_members;
  a.S = p->num_seqs;
  a.Hkv = p->num_kv_heads;
  a.G = p->num_q_heads / p->num_kv_heads;
  a.nb = p->num_blocks;
  a.max_ctx = p->max_context;
  a.log_b = p->block_size == 16 ? 4 : p->block_size == 32 ? 5 : 6;
  a.tile_rows = l.tile_rows;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.st_o = (float*)p->workspace;
  a.st_ml = (float2*)((char*)p->workspace + w.ml);
  const dim3 grid((unsigned)(l.num_items + (l.num_pieces + kPrefixWaves - 1) / kPrefixWaves));
  hipStream_t st = (hipStream_t)stream;
  if (p->head_dim == 64) {
    if (int8) launch_prefix<64, 1>(l.tile_rows, grid, st, a);
    else launch_prefix<64, 0>(l.tile_rows, grid, st, a);
  } else {
    if (int8) launch_prefix<128, 1>(l.tile_rows, grid, st, a);
    else launch_prefix<128, 0>(l.tile_rows, grid, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "prefix attention launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}
