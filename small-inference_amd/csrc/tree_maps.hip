// Drafted trees around a forward: its metadata built on the device from the sequences' lengths and the nodes' parents,
// and, once the forward has been verified, the accepted nodes' K and V moved to the positions they now have.
//
// The reference decodes one token per step and has neither; slots, positions and packed tables follow the rules of its
// engine/paged_cache.py:55-90 and engine/block_manager.py:118-123.
#include "sipa_common.h"

namespace sipa {

constexpr int kTreeMaxSeqs = 8192;  // query starts of all sequences in LDS: 32 KB

struct TreeMapsArgs {
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_rows, table_width;
  const int32_t* rows;
  const int32_t* starts;
  const int32_t* counts;
  const int32_t* parents;
  int32_t S, T, B, W, words;
  int32_t token_groups;  // workgroups of 256 nodes; the ones behind them take 256 entries of the packed tables each
  int64_t* positions;
  int64_t* slots;
  int64_t* slot_blocks;
  int64_t* slot_offsets;
  int64_t* last_rows;
  int32_t* query_starts;
  int32_t* ctx;
  int32_t* bt;
  uint64_t* ancestors;
  bool fill_rest;
  int64_t rest_slot;
};

__device__ __forceinline__ int32_t tree_table_entry(const TreeMapsArgs& a, int s, int64_t col) {
  const int row = min(max(a.rows[s], 0), a.table_rows - 1);
  const int c = (int)min(max(col, (int64_t)0), (int64_t)a.table_width - 1);
  return a.tables[(int64_t)row * a.table_stride + c];
}

// Every workgroup forms the query starts for itself (S loads that the L2 serves, one scan), so that one launch does it all: bound
// by the latency of its chain of loads, not by bytes: 3.5 us for 1 tree of 5 nodes; 9.1 us for 256 ragged trees of up to 64
// nodes at 8192 tokens. An ancestor is one load after the other, as many as the tree is deep.
__global__ void __launch_bounds__(256) tree_maps_kernel(const TreeMapsArgs a) {
  __shared__ int32_t qs[kTreeMaxSeqs + 1];
  __shared__ int32_t part[256];
  const int tid = threadIdx.x;
  const int per = (a.S + 255) / 256, s0 = min(tid * per, a.S), s1 = min(s0 + per, a.S);
  int64_t sum = 0;
  for (int s = s0; s < s1; ++s) sum += max(a.counts[s], 0);
  part[tid] = (int32_t)min(sum, (int64_t)a.T);
  __syncthreads();
  for (int d = 1; d < 256; d *= 2) {  // inclusive sums, saturating at T
    const int32_t x = tid >= d ? part[tid - d] : 0;
    __syncthreads();
    part[tid] = (int32_t)min((int64_t)part[tid] + x, (int64_t)a.T);
    __syncthreads();
  }
  int64_t at = tid ? part[tid - 1] : 0;
  for (int s = s0; s < s1; ++s) {
    qs[s] = (int32_t)at;
    at = min(at + max(a.counts[s], 0), (int64_t)a.T);
  }
  if (tid == 255) qs[a.S] = part[255];
  __syncthreads();
  if ((int)blockIdx.x < a.token_groups) {
    const int t = (int)blockIdx.x * 256 + tid;
    if (t >= qs[a.S]) {
      if (!a.fill_rest || t >= a.T) return;
      for (int w = 0; w < a.words; ++w) a.ancestors[(int64_t)t * a.words + w] = 0;
      a.positions[t] = 0;
      a.slots[t] = a.rest_slot;
      a.slot_blocks[t] = a.rest_slot / a.B;
      a.slot_offsets[t] = a.rest_slot % a.B;
      return;
    }
    int lo = 0, hi = a.S;  // the last s with qs[s] <= t: sequences without nodes share their successor's start
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (qs[mid] <= t) lo = mid; else hi = mid;
    }
    const int s = lo, first = qs[s], i = t - first;
    uint64_t bits[4] = {0, 0, 0, 0};
    int depth = -1;
    for (int node = i; node >= 0;) {
      if (node < 256) bits[node >> 6] |= 1ull << (node & 63);
      ++depth;
      const int up = a.parents[first + node];
      node = up < node ? up : -1;
    }
    for (int w = 0; w < a.words; ++w) a.ancestors[(int64_t)t * a.words + w] = bits[w];
    const int64_t p = (int64_t)a.starts[s] + i;
    const int64_t blk = tree_table_entry(a, s, p / a.B);
    a.positions[t] = (int64_t)a.starts[s] + depth;
    a.slots[t] = blk * a.B + p % a.B;
    a.slot_blocks[t] = blk;
    a.slot_offsets[t] = p % a.B;
    return;
  }
  const int64_t j = ((int64_t)blockIdx.x - a.token_groups) * 256 + tid;
  if (j >= (int64_t)a.S * a.W) return;
  const int s = (int)(j / a.W), c = (int)(j % a.W);
  const int64_t ctx = (int64_t)a.starts[s] + (qs[s + 1] - qs[s]);
  a.bt[j] = (int64_t)c * a.B < ctx ? tree_table_entry(a, s, c) : -1;
  if (c == 0) {
    a.ctx[s] = (int32_t)ctx;
    a.last_rows[s] = (int64_t)qs[s + 1] - 1;
    a.query_starts[s] = qs[s];
    if (s == 0) a.query_starts[a.S] = qs[a.S];
  }
}

struct CommitArgs {
  uint8_t* pool[2];
  int64_t sl[2], sh[2];
  uint16_t* scale[2];
  int64_t ssl[2], ssh[2];
  const int32_t* bt;
  int64_t bt_ss;
  const int32_t* starts;
  const int32_t* accepted;
  int64_t acc_ss;
  const int32_t* num;
  int32_t L, H, N, B, row_bytes, S, A, W;
  int32_t parts;  // threads of a (pool, layer, head, sequence): 16-byte parts of a row, then one for the scales
  int64_t threads;
};

// One thread takes one 16-byte part of the moved rows of a (sequence, pool, layer, head), all its moves in order: source
// indices ascend and are at least their destinations', so a load never reads what an earlier store has written. Kept at
// kMoves loads in flight before their stores: 4.4 us for up to 4 nodes of one sequence in 24 layers, a short chain of loads
// (index, block id, row); 10.7 us for 64 sequences' up to 7 nodes in 28 layers of INT8 pools, where the 64-bit divisions by
// the block size, two a move, and by the thread's dimensions weigh more than the 1.6 us of bytes (a call with the host's part:
// 8.0 and 11.9).
constexpr int kMoves = 8;

__global__ void __launch_bounds__(256) commit_tokens_kernel(const CommitArgs a) {
  int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.threads) return;
  const int part = (int)(i % a.parts);
  i /= a.parts;
  const int h = (int)(i % a.H);
  i /= a.H;
  const int l = (int)(i % a.L);
  i /= a.L;
  const int kv = (int)(i & 1), s = (int)(i >> 1);
  const int n = min(max(a.num[s], 0), a.A);
  const int64_t start = a.starts[s];
  const int32_t* acc = a.accepted + (int64_t)s * a.acc_ss;
  const int32_t* table = a.bt + (int64_t)s * a.bt_ss;
  const int64_t top = (int64_t)a.W * a.B - 1;
  auto slot = [&](int64_t p) {
    p = min(max(p, (int64_t)0), top);
    return (int64_t)min(max(table[p / a.B], 0), a.N - 1) * a.B + p % a.B;
  };
  const bool scales = part * 16 >= a.row_bytes;
  uint8_t* pool = a.pool[kv] + l * a.sl[kv] + h * a.sh[kv] + 16 * part;
  uint16_t* sp = scales ? a.scale[kv] + l * a.ssl[kv] + h * a.ssh[kv] : nullptr;
  for (int b = 0; b < n; b += kMoves) {
    uint4 x[kMoves];
    uint16_t y[kMoves];
    int64_t to[kMoves];
#pragma unroll
    for (int u = 0; u < kMoves; ++u) {
      const int m = b + u;
      to[u] = -1;
      if (m >= n || acc[m] == m) continue;
      const int64_t from = slot(start + acc[m]);
      to[u] = slot(start + m);
      if (scales) y[u] = sp[from];
      else x[u] = *(const uint4*)(pool + from * a.row_bytes);
    }
#pragma unroll
    for (int u = 0; u < kMoves; ++u) {
      if (to[u] < 0) continue;
      if (scales) sp[to[u]] = y[u];
      else *(uint4*)(pool + to[u] * a.row_bytes) = x[u];
    }
  }
}

}  // namespace sipa

using namespace sipa;

extern "C" int32_t sipa_tree_maps(const sipa_tree_maps_params* p, void* stream) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_tree_maps_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_tree_maps_params (%d bytes)",
             (int)sizeof(sipa_tree_maps_params));
  SIPA_CHECK(p->num_seqs > 0 && p->num_seqs <= kTreeMaxSeqs && p->num_tokens > 0, SIPA_EINVAL,
             "%d sequences (1 .. %d), %d nodes", p->num_seqs, kTreeMaxSeqs, p->num_tokens);
  SIPA_CHECK(p->words >= 1 && p->words <= 4, SIPA_EINVAL, "%d mask words (1 .. 4)", p->words);
  SIPA_CHECK(p->block_size > 0 && p->out_width > 0 && p->table_rows > 0 && p->table_width > 0 &&
                 p->table_stride >= p->table_width, SIPA_EINVAL, "bad table or block sizes");
  SIPA_CHECK(p->tables && p->rows && p->starts && p->counts && p->parents && p->positions && p->slots &&
                 p->slot_blocks && p->slot_offsets && p->last_rows && p->query_starts && p->context_lens &&
                 p->block_tables && p->ancestors, SIPA_EINVAL, "NULL pointer");
  SIPA_CHECK(!p->fill_rest || p->rest_slot >= 0, SIPA_EINVAL, "slot %lld for the rows behind", (long long)p->rest_slot);
  TreeMapsArgs a;
  a.fill_rest = p->fill_rest != 0;
  a.rest_slot = p->rest_slot;
  a.tables = p->tables;
  a.table_stride = p->table_stride;
  a.table_rows = p->table_rows;
  a.table_width = p->table_width;
  a.rows = p->rows;
  a.starts = p->starts;
  a.counts = p->counts;
  a.parents = p->parents;
  a.S = p->num_seqs;
  a.T = p->num_tokens;
  a.B = p->block_size;
  a.W = p->out_width;
  a.words = p->words;
  a.token_groups = (int32_t)(((int64_t)p->num_tokens + 255) / 256);
  a.positions = p->positions;
  a.slots = p->slots;
  a.slot_blocks = p->slot_blocks;
  a.slot_offsets = p->slot_offsets;
  a.last_rows = p->last_rows;
  a.query_starts = p->query_starts;
  a.ctx = p->context_lens;
  a.bt = p->block_tables;
  a.ancestors = p->ancestors;
  const int64_t grid = a.token_groups + ((int64_t)a.S * a.W + 255) / 256;
  SIPA_CHECK(grid <= 0x7fffffff, SIPA_EINVAL, "tree maps grid too large");
  hipLaunchKernelGGL(tree_maps_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "tree maps launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}

extern "C" int32_t sipa_commit_tokens(const sipa_commit_params* p, void* stream) {
  SIPA_CHECK(p != nullptr && p->struct_size == (int32_t)sizeof(sipa_commit_params), SIPA_EINVAL,
             "struct_size does not match this library's sipa_commit_params (%d bytes)",
             (int)sizeof(sipa_commit_params));
  SIPA_CHECK(p->num_layers > 0 && p->num_kv_heads > 0 && p->num_blocks > 0 && p->block_size > 0 && p->num_seqs >= 0 &&
                 p->max_accepted >= 0 && p->bt_width > 0, SIPA_EINVAL, "bad pool or sequence sizes");
  SIPA_CHECK(p->row_bytes > 0 && p->row_bytes % 16 == 0, SIPA_EUNSUPPORTED, "rows of %d bytes (a multiple of 16)",
             p->row_bytes);
  if (p->num_seqs == 0 || p->max_accepted == 0) return SIPA_OK;
  SIPA_CHECK(p->k_pool && p->v_pool && p->block_tables && p->starts && p->accepted && p->num_accepted, SIPA_EINVAL,
             "NULL pointer");
  SIPA_CHECK((p->k_scale == nullptr) == (p->v_scale == nullptr), SIPA_EINVAL, "scales of K and V go together");
  SIPA_CHECK((((uintptr_t)p->k_pool | (uintptr_t)p->v_pool | (uint64_t)p->k_stride_l | (uint64_t)p->k_stride_h |
               (uint64_t)p->v_stride_l | (uint64_t)p->v_stride_h) & 15) == 0, SIPA_EINVAL,
             "pools and their strides must be 16-byte aligned");
  CommitArgs a;
  a.pool[0] = (uint8_t*)p->k_pool;
  a.pool[1] = (uint8_t*)p->v_pool;
  a.sl[0] = p->k_stride_l, a.sl[1] = p->v_stride_l;
  a.sh[0] = p->k_stride_h, a.sh[1] = p->v_stride_h;
  a.scale[0] = (uint16_t*)p->k_scale;
  a.scale[1] = (uint16_t*)p->v_scale;
  a.ssl[0] = p->ks_stride_l, a.ssl[1] = p->vs_stride_l;
  a.ssh[0] = p->ks_stride_h, a.ssh[1] = p->vs_stride_h;
  a.bt = p->block_tables;
  a.bt_ss = p->bt_stride_s;
  a.starts = p->starts;
  a.accepted = p->accepted;
  a.acc_ss = p->acc_stride_s;
  a.num = p->num_accepted;
  a.L = p->num_layers;
  a.H = p->num_kv_heads;
  a.N = p->num_blocks;
  a.B = p->block_size;
  a.row_bytes = p->row_bytes;
  a.S = p->num_seqs;
  a.A = p->max_accepted;
  a.W = p->bt_width;
  a.parts = p->row_bytes / 16 + (p->k_scale != nullptr);
  a.threads = 2ll * a.S * a.L * a.H * a.parts;
  const int64_t grid = (a.threads + 255) / 256;
  SIPA_CHECK(grid <= 0x7fffffff, SIPA_EINVAL, "commit grid too large");
  hipLaunchKernelGGL(commit_tokens_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIPA_EHIP, "commit launch failed: %s", hipGetErrorString(e));
  return SIPA_OK;
}
