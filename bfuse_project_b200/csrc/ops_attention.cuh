// Attention over packed sequences on sm_100a: out = softmax(scale * q k^T) v, causal or not, grouped
// heads, in one pass over the keys.  The three steps that bfuse_project_b200/attention.py chains
// through score matrices in memory (the reference's bgemm_0 / softmax / bgemm_1,
// test-utils/examples/llm.yaml:38-49) stay on the chip here: per 128 keys
//
//     S = Q K^T                                   tcgen05, operands in shared memory, fp32 in tensor memory
//     m' = max(m, max_j S), p = 2^(c (S - m'))    c = scale * log2(e); one thread per row
//     l' = l 2^(c (m - m')) + sum_j p
//     O' = O 2^(c (m - m')) + p V                 tcgen05, p as bf16 in tensor memory, O fp32 in tensor memory
//
// and out = O / l at the end.
//
// A tile is 128 rows of queries that share one key / value head: P = 128 / G consecutive positions of
// one sequence times the G query heads of the group, so a single token of a grouped model fills G rows
// and a prompt's tile reads each key once for the whole group.  BlockDim = (192, 1, 1): warps 0-3 own
// the rows (thread = row = lane of tensor memory), warp 4 issues the TMA loads, warp 5 the MMAs.  (Eight
// warps, two threads a row, are no faster: the two have to exchange their maxima in every block.  Nor are
// polynomials for an eighth to a half of the exponentials: what MUFU saves, their instructions cost.)
// GridDim = (slices * kv heads, tiles); the tiles are counted from the sequence offsets on the device
// (`find_tile`), the host knows only their number at most: (total_q + seqs (P - 1)) / P.  The last
// tile of a sequence, the one with the most keys under a causal mask, comes first.
//
// Few rows over many keys: the `slices` CTAs of a tile form a thread-block cluster, each takes a run of
// its 128-key blocks, and they join through distributed shared memory as the k-slices of the GEMM body
// do -- first every rank's (m, l) of every row, then its O scaled by 2^(m_rank - m) / l, summed in rank
// order by the rank that owns the columns (deterministic).
//
// A tile of at most 16 rows (single tokens) would leave most of those exponentials to rows that are not
// there.  It is multiplied the other way round: S^T = K Q^T and O^T += V^T p^T, keys (then dims) in the
// lanes and the rows in 16 columns; a thread owns a key, p^T goes through shared memory, and S of the next
// block is made while this one's exponentials are taken.
//
// Many short tiles: a CTA that is through its tile takes that of a block that has not started (clusterlaunchcontrol), whose keys
// are loaded meanwhile; barriers and tensor memory stay.  A block of its own costs 7 us a tile of one block of keys, 3.6 of
// them beside another CTA's; a walk's tile 2.9.
//
// What bounds it: long prompts the softmax between the MMAs of two tiles (a pair of blocks of 128 dims takes 3600 clocks, 2048 of
// MMAs and 2048 of exponentials) and the power the device may draw; single tokens the loads of the CTA with the longest run of keys.
//
// Tensor memory: S in columns 0-127, O in columns 128 up, the bf16 p in 64 columns of its own behind O where
// there is room (heads of up to 64 in 256 columns; 512 columns where only one CTA fits an SM anyway), else over S.
// Two CTAs of 256 columns share an SM, and one's MMAs run under the other's exponentials.
#pragma once

#include "ops_umma.cuh"

namespace bfuse {

__host__ __device__ constexpr int attn_threads(int tiles) { return 128 * tiles + 64; }
constexpr int kAttnRows = 128;     // query rows of a tile
constexpr int kAttnKeys = 128;     // keys of a block
constexpr int kAttnChunkBytes = 128 * 128;   // 128 rows x 64 bf16: what one TMA box holds
constexpr int kAttnFewRows = 16;   // tiles of at most so many rows run transposed
constexpr int kAttnMaxStages = 8;

enum AttnStatus : int {
  ATTN_WAIT_Q_TIMEOUT = 0x301,
  ATTN_WAIT_KV_TIMEOUT = 0x302,
  ATTN_WAIT_SLOT_TIMEOUT = 0x303,
  ATTN_WAIT_SCORES_TIMEOUT = 0x304,
  ATTN_WAIT_PROBS_TIMEOUT = 0x305,
  ATTN_WAIT_OUT_TIMEOUT = 0x306,
  ATTN_WAIT_PEERS_TIMEOUT = 0x307,
  ATTN_WAIT_TILE_TIMEOUT = 0x308,
  ATTN_BAD_OFFSETS = -1,   // BFUSE_STATUS_BAD_OFFSETS: sequence offsets that fall, or that leave the tensors: that sequence is left out
};

__host__ __device__ constexpr int attn_chunks(int dim) { return dim <= 64 ? 1 : 2; }   // 64-element chunks of a head
__host__ __device__ constexpr int attn_tile_bytes(int dim) { return attn_chunks(dim) * kAttnChunkBytes; }
// behind the ring, with key slices: what the ranks push to one another for a tile of few rows, (m, l) of 16 rows from each of up
// to 8 and 128 dims of 16 rows
constexpr int kAttnFewStats = 8 * 16 * 8;
__host__ __device__ constexpr int attn_few_join_bytes(int split) { return split > 1 ? kAttnFewStats + 128 * 16 * 4 : 0; }
__host__ __device__ constexpr int attn_smem_bytes(int dim, int tiles, int stages, int split) {
  return kUmmaHeaderBytes + (tiles + stages) * attn_tile_bytes(dim) + attn_few_join_bytes(split);
}
// what the slices of a whole tile exchange at the end, over Q and the ring: (m, l) per rank and row, and per 16 owned columns 8 KB of every rank
__host__ __device__ constexpr int attn_join_bytes(int dim, int split) {
  return split > 1 ? split * kAttnRows * 8 + ((attn_chunks(dim) * 4 + split - 1) / split) * split * 16 * kAttnRows * 4 : 0;
}

struct AttentionParams {
  alignas(64) CUtensorMap map_q;   // {dim, query heads, tokens}, box {64, group, positions}, 128B swizzle
  alignas(64) CUtensorMap map_k;   // {dim, kv heads, tokens}, box {64, 1, 128}, 128B swizzle
  alignas(64) CUtensorMap map_v;
  const int *cu_q, *cu_kv;         // [seqs + 1] first token of every sequence, and the end of the last
  uint16_t *out;                   // [total_q, heads, dim]
  int seqs, total_q, total_kv, heads, kv_heads, dim;
  int group, positions;            // query heads per kv head; positions of a tile
  int causal, split, stages;
  int sort;                        // longest sequences first
  int tmem_cols, p_col;            // tensor memory: columns in all; first column of p, 0: over the scores
  float scale_log2;                // scale * log2(e), positive
};

// 32 lanes x 32 consecutive fp32 columns: thread i of the warp gets lane i; valid after tmem_ld_wait()
__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// registers -> 32 lanes x 16 columns; complete after tmem_st_wait()
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D += A B with A (bf16, two values a column) in tensor memory and B in shared memory
__device__ __forceinline__ void umma_ts_bf16(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 8-byte store into a peer's shared memory that also credits 8 bytes to the peer's mbarrier
__device__ __forceinline__ void st_async_f2(uint32_t peer_addr, uint32_t peer_bar, float a, float b) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%2, %3}, [%1];" ::"r"(peer_addr), "r"(peer_bar),
               "r"(__float_as_uint(a)), "r"(__float_as_uint(b))
               : "memory");
}
__device__ __forceinline__ float2 ld_shared_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// One tile of queries, as find_tile leaves it in shared memory.
struct AttnTile {
  int found;      // 0: this block has no tile, -1: a walk ends here
  int head;       // kv head
  int q0, npos;   // first token, positions (<= P) of the tile
  int kv0, kv_len;
  int last0;      // causal: key index (within the sequence) that the tile's first position may see last
  int keys;       // keys that any row of the tile may see
  // what came before it in a walk, which says the phase a barrier is in: loads of the ring and of queries; blocks of keys, by tile
  // of the CTA (one tile: whole tiles, and tiles of few rows); tiles with keys
  uint32_t loads, queries, blocks[2], outs[2];
};

// ---- a walk: the CTA asks for the number of a block that has not started, which then never starts ----
__device__ __forceinline__ void ask_block(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
// -1: every block has started
__device__ __forceinline__ int answered_block(uint32_t answer) {
  int block;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\tld.shared.b128 a, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tmov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, a;\n\t}"
      : "=r"(block)
      : "r"(answer)
      : "memory");
  return block;
}

// T tiles of one sequence and kv head per CTA: 1, or 2 that share every block of keys (four more warps; whole tiles only).
// WALK: a CTA that is through its tile goes on with that of a block that has not started yet, whose keys are loaded meanwhile
// (alone in its launch, one key slice).
template <int T, bool WALK>
struct Attention {
  using Params = AttentionParams;
  static constexpr int kMaxThreads = attn_threads(T);
  static constexpr int kMinBlocks = T == 1 ? 2 : 1;   // two CTAs an SM: 168 registers a thread, 128 of them a row's scores
  static constexpr bool kMemoryBound = false;
  static constexpr bool kUsesTmem = true;
  static constexpr int kProducer = 4 * T, kIssuer = kProducer + 1;   // warps

  // The window: [0, 1024) barriers, tensor-memory pointer and the tile; [1024, 2048) what the threads of a row exchange;
  // then Q and the ring of `stages` K / V blocks in the order K0 V0 K1 V1 ...
  struct Window {
    // s_bar, pv_bar, o_bar, c_bar: one per tile, p_bar: two per tile; few rows: two sf_bar and pf_bar, by the parity of the block;
    // a walk: tile_bar, the next tile is known, done_bar, all are through one (two each, by the tile's parity: whoever is quick may
    // be a tile ahead of whoever waits), next_bar, the answer is there
    uint32_t full0, empty0, q_bar, s_bar, p_bar, pv_bar, o_bar, c_bar, stats_bar, join_bar, sf_bar, pf_bar, pvf_bar, tile_bar, done_bar, next_bar, next;
    uint32_t xch, q, ring, few_join;
    int chunks, tile_bytes;
  };
  static constexpr int kBars = 2 * kAttnMaxStages + 25;

  // Tile number t of the batch (T = 2: pair of tiles) into *tile: sequence i has ceil(len_i / (T P)) of them, the last
  // positions first.  One warp.  Up to 32 sequences: one a lane, the longest first where `sort` (more tiles than run at
  // once: a long sequence that starts late ends last); more: 256 a round, 8 a lane (the last of the `tiles` there may be looks
  // at every sequence, so that bad offsets are seen even if no tile is theirs).
  __device__ __forceinline__ static void find_tile(const Params &p, int t, int tiles, int lane, AttnTile *tile, int *status) {
    const int positions = T * p.positions;
    auto bad = [&] { atomicCAS(status, 0, (int)ATTN_BAD_OFFSETS); };
    auto put = [&](int q0, int q_len, int kv0, int kv_end, int qt) {
      AttnTile r = *tile;   // (head, and what came before)
      r.found = kv0 >= 0 && kv_end >= kv0 && kv_end <= p.total_kv;
      if (!r.found) bad();
      r.q0 = q0 + qt * positions;
      r.npos = min(positions, q_len - qt * positions);
      r.kv0 = kv0;
      r.kv_len = kv_end - kv0;
      r.last0 = r.kv_len - q_len + qt * positions;
      r.keys = p.causal ? max(0, min(r.kv_len, r.last0 + r.npos)) : r.kv_len;
      *tile = r;
    };
    if (lane == 0) tile->found = 0;
    __syncwarp();
    if (p.seqs <= 32) {
      const int s0 = min(lane, p.seqs);
      const int qa = __ldg(p.cu_q + s0), ka = __ldg(p.cu_kv + s0), qb = __ldg(p.cu_q + min(s0 + 1, p.seqs)), kb = __ldg(p.cu_kv + min(s0 + 1, p.seqs));
      int n = 0;
      if (lane < p.seqs) {
        if (qa < 0 || qb < qa || qb > p.total_q) bad();
        else n = (qb - qa + positions - 1) / positions;
      }
      int at = 0;   // first tile of this lane's sequence
      if (p.sort) {
        const int len = qb - qa + (kb - ka);
        for (int i = 0; i < p.seqs; ++i) {
          const int m = __shfl_sync(0xffffffffu, n, i), other = __shfl_sync(0xffffffffu, len, i);
          if (other > len || (other == len && i < lane)) at += m;
        }
      } else {
        int upto = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, off);
          if (lane >= off) upto += v;
        }
        at = upto - n;
      }
      if (t >= at && t < at + n) put(qa, qb - qa, ka, kb, n - 1 - (t - at));
      __syncwarp();
      return;
    }
    int before = 0;   // tiles of the sequences before this round's
    for (int base = 0; base < p.seqs; base += 256) {
      const int s0 = base + lane * 8;
      int cu[9], n[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 9; ++i) cu[i] = __ldg(p.cu_q + min(s0 + i, p.seqs));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] = 0;
        if (s0 + i < p.seqs) {
          if (cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > p.total_q) bad();
          else n[i] = (cu[i + 1] - cu[i] + positions - 1) / positions;
        }
        mine += n[i];
      }
      int upto = mine;   // inclusive sum over the lanes
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += v;
      }
      const int total = __shfl_sync(0xffffffffu, upto, 31);
      if (t - before < total) {
        int at = before + upto - mine;   // first tile of this lane's sequences
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (t >= at && t < at + n[i]) put(cu[i], cu[i + 1] - cu[i], __ldg(p.cu_kv + s0 + i), __ldg(p.cu_kv + s0 + i + 1), n[i] - 1 - (t - at));
          at += n[i];
        }
        __syncwarp();
        if (t + 1 < tiles) return;
      }
      before += total;
    }
  }

  __device__ __forceinline__ static Window window(const Params &p, uint32_t base) {
    Window w;
    w.full0 = base, w.empty0 = w.full0 + 8 * kAttnMaxStages, w.q_bar = w.empty0 + 8 * kAttnMaxStages;
    w.s_bar = w.q_bar + 8, w.p_bar = w.q_bar + 24, w.pv_bar = w.q_bar + 56, w.o_bar = w.q_bar + 72, w.c_bar = w.q_bar + 88, w.stats_bar = w.q_bar + 104, w.join_bar = w.q_bar + 112;
    w.sf_bar = w.q_bar + 120, w.pf_bar = w.q_bar + 136, w.pvf_bar = w.q_bar + 152, w.tile_bar = w.q_bar + 160, w.done_bar = w.q_bar + 176, w.next_bar = w.q_bar + 192;
    w.next = w.full0 + 768, w.xch = w.full0 + 1024, w.q = w.full0 + kUmmaHeaderBytes;
    w.chunks = attn_chunks(p.dim), w.tile_bytes = w.chunks * kAttnChunkBytes, w.ring = w.q + T * w.tile_bytes, w.few_join = w.ring + p.stages * w.tile_bytes;
    return w;
  }

  // arrivals at barrier i from q_bar on: the 128 threads of a tile at p_bar (four), c_bar and pf_bar (two each), those of every
  // tile and the issuer at done_bar
  __device__ __forceinline__ static int arrivals(const Window &w, int i) {
    const uint32_t bar = w.q_bar + 8 * i;
    if (bar == w.done_bar || bar == w.done_bar + 8) return 128 * T + 1;
    return (bar >= w.p_bar && bar < w.pv_bar) || (bar >= w.c_bar && bar < w.stats_bar) || (bar >= w.pf_bar && bar < w.pvf_bar) ? 128 : 1;
  }
  // what came before a tile
  __device__ __forceinline__ static uint32_t loads(const AttnTile &t) { return WALK ? t.loads : 0u; }
  __device__ __forceinline__ static uint32_t blocks(const AttnTile &t, int x) { return WALK ? t.blocks[x] : 0u; }
  __device__ __forceinline__ static uint32_t outs(const AttnTile &t, int x) { return WALK ? t.outs[x] : 0u; }

  // this slice's blocks of keys: first and count
  __device__ __forceinline__ static void my_blocks(const AttnTile &t, int split, int slice, int &b0, int &n) {
    const int nblocks = (t.keys + kAttnKeys - 1) / kAttnKeys, per = (nblocks + split - 1) >> log2_of(split);   // (a power of two)
    b0 = min(nblocks, slice * per);
    n = min(nblocks, b0 + per) - b0;
  }
  __device__ __forceinline__ static bool few_rows(const Params &p, const AttnTile &t) { return T == 1 && t.npos * p.group <= kAttnFewRows; }
  // tile x of the CTA's, and its blocks of keys (those that some row of it may see come first in the CTA's n)
  __device__ __forceinline__ static AttnTile sub_tile(const Params &p, const AttnTile &t, int x) {
    if (T == 1) return t;
    AttnTile s = t;
    s.npos = max(0, min(p.positions, t.npos - x * p.positions));
    s.q0 += x * p.positions;
    s.last0 += x * p.positions;
    s.keys = s.npos == 0 ? 0 : p.causal ? max(0, min(s.kv_len, s.last0 + s.npos)) : s.kv_len;
    return s;
  }
  __device__ __forceinline__ static int sub_blocks(const AttnTile &s, int n) { return T == 1 ? n : (s.keys + kAttnKeys - 1) / kAttnKeys; }

  // load i of the ring: K or V of block i / 2
  __device__ __forceinline__ static void load(const Params &p, const Window &w, const AttnTile &t, int b0, int i, uint32_t slot) {
    const uint32_t bar = w.full0 + 8 * slot, dst = w.ring + slot * w.tile_bytes;
    const int token = t.kv0 + (b0 + (i >> 1)) * kAttnKeys;
    const CUtensorMap *map = i & 1 ? &p.map_v : &p.map_k;
    mbar_expect_tx(bar, (uint32_t)w.tile_bytes);
    for (int ch = 0; ch < w.chunks; ++ch) tma_load_3d(dst + ch * kAttnChunkBytes, map, bar, ch * 64, t.head, token);
  }

  // 16 finished columns of a row
  __device__ __forceinline__ static void store16(uint16_t *row, int col, int dim, const float (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (col + 8 * j < dim)
        *reinterpret_cast<uint4 *>(row + col + 8 * j) = make_uint4(f2_to_bf16x2(v[8 * j], v[8 * j + 1]), f2_to_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                                                                   f2_to_bf16x2(v[8 * j + 4], v[8 * j + 5]), f2_to_bf16x2(v[8 * j + 6], v[8 * j + 7]));
  }
  // element 0 of a row of the tile in out
  __device__ __forceinline__ static uint16_t *out_row(const Params &p, const AttnTile &t, int head, int row) {
    const int pos = row / p.group;
    return p.out + ((size_t)(t.q0 + pos) * p.heads + head * p.group + (row - pos * p.group)) * p.dim;
  }

  // (of a tile that some row sees keys of.  Two tiles: the first may be without, when the causal mask hides every key from it; its
  // threads wait for nothing and stage their zeros where its queries would be)
  __device__ __forceinline__ static void load_q(const Params &p, const Window &w, const AttnTile &t) {
    const int tiles = T == 2 && t.npos > p.positions ? 2 : 1, first = T == 2 && sub_tile(p, t, 0).keys == 0 ? 1 : 0;
    mbar_expect_tx(w.q_bar, (uint32_t)((tiles - first) * w.chunks * p.group * p.positions * 128));
    for (int x = first; x < tiles; ++x)
      for (int ch = 0; ch < w.chunks; ++ch)
        tma_load_3d(w.q + x * w.tile_bytes + ch * kAttnChunkBytes, &p.map_q, w.q_bar, ch * 64, t.head * p.group, t.q0 + x * p.positions);
  }
  // loads [from, to) of a tile, each once its slot of the ring is free
  __device__ __forceinline__ static bool load_run(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int b0, int from, int to) {
    const uint32_t stages = (uint32_t)p.stages, at = loads(t) + (uint32_t)from;
    uint32_t s = at % stages, round = at / stages;
    for (int i = from; i < to; ++i) {
      if (round > 0 && !mbar_wait(w.empty0 + 8 * s, (round - 1) & 1, c.status, ATTN_WAIT_SLOT_TIMEOUT)) return false;
      load(p, w, t, b0, i, s);
      if (++s == stages) s = 0, ++round;
    }
    return true;
  }

  // The loading warp of a walk.  With a tile's last load on its way it asks for the next tile, finds it and loads what the ring has
  // room for of its keys; the queries wait until everyone is through the tile before.
  __device__ __forceinline__ static void lead(const Params &p, const TileCtx &c, const Window &w, AttnTile *tile_slot, int loaded, int lane) {
    AttnTile t = tile_slot[0];
    bool ok = true;
    for (int i = 0;; ++i) {
      int b0 = 0, n = 0;
      if (t.found) my_blocks(t, 1, 0, b0, n);
      if (elect_one()) {
        ok = load_run(p, c, w, t, b0, loaded, 2 * n);
        mbar_expect_tx(w.next_bar, 16);
        ask_block(w.next, w.next_bar);
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, ok);
      ok = warp_wait(w.next_bar, i & 1, c.status, ATTN_WAIT_TILE_TIMEOUT) && ok;
      const int block = ok ? answered_block(w.next) : -1;
      fence_async_smem();   // (it has been read: the next one may be written)
      AttnTile *slot = tile_slot + ((i + 1) & 1);   // everyone is through tile i - 1
      if (lane == 0) {
        t.loads += 2 * n;
        t.queries += n > 0;
        for (int x = 0; x < 2; ++x) {
          const int nx = T == 2 ? (n > 0 ? sub_blocks(sub_tile(p, t, x), n) : 0) : few_rows(p, t) == (x == 1) ? n : 0;
          t.blocks[x] += nx;
          t.outs[x] += T == 2 ? nx > 0 : n > 0;
        }
        t.head = block < 0 ? 0 : block % c.gx;
        t.found = block < 0 ? -1 : 0;
        *slot = t;
      }
      __syncwarp();
      if (block >= 0) find_tile(p, block / c.gx, c.gy, lane, slot, c.status);
      __syncwarp();
      if (lane == 0) mbar_arrive(w.tile_bar + 8 * ((i + 1) & 1));
      if (block < 0) return;
      t = *slot;
      n = 0;
      if (t.found) my_blocks(t, 1, 0, b0, n);
      loaded = min(p.stages, 2 * n);
      if (elect_one()) {
        ok = load_run(p, c, w, t, b0, 0, loaded);
        ok = mbar_wait(w.done_bar + 8 * (i & 1), (i >> 1) & 1, c.status, ATTN_WAIT_TILE_TIMEOUT) && ok;
        if (ok && n > 0) load_q(p, w, t);
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, ok);
    }
  }

  // The issuing warp's part of a tile
  __device__ __forceinline__ static void issue(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int b0, int n, bool few, uint32_t tmem) {
    const int stages = p.stages;
    if (n > 0 && elect_one()) {
      bool ok = mbar_wait(w.q_bar, WALK ? t.queries & 1 : 0, c.status, ATTN_WAIT_Q_TIMEOUT);
      if (ok) ok = few ? multiply_few(p, c, w, t, n, tmem) : multiply(p, c, w, t, n, tmem);
      if (T == 1) umma_commit(w.o_bar);
      // the releases of the slots' last uses are asynchronous: none may be in flight when the barriers go
      for (int i = max(0, 2 * n - stages); i < 2 * n && ok; ++i) {
        const uint32_t at = loads(t) + (uint32_t)i;
        ok = mbar_wait(w.empty0 + 8 * (at % (uint32_t)stages), (at / (uint32_t)stages) & 1, c.status, ATTN_WAIT_SLOT_TIMEOUT);
      }
      for (int x = 0; x < T && ok; ++x) {
        const int nx = sub_blocks(sub_tile(p, t, x), n);
        if (nx > 0 && few) ok = mbar_wait(w.pvf_bar, (blocks(t, 1) + nx - 1) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
        if (nx > 0 && !few && p.p_col) ok = mbar_wait(w.pv_bar + 8 * x, (blocks(t, x) + nx - 1) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
        if (nx > 0 && ok) ok = mbar_wait(w.o_bar + 8 * x, outs(t, x) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
      }
    }
    __syncwarp();
  }
  // The other warps' part (with key slices, where all of them meet the cluster's, every warp's)
  __device__ __forceinline__ static void rows(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int split, int slice, int b0, int n, bool few, uint32_t tmem) {
    const int warp = c.tid >> 5;
    if constexpr (T == 2) {
      const AttnTile s = sub_tile(p, t, warp >> 2);
      tile(p, c, w, s, t.head, 1, 0, 0, sub_blocks(s, n), tmem, warp >> 2);
    } else if (few) {
      if (t.npos * p.group <= 8) few_tile<8>(p, c, w, t, t.head, split, slice, b0, n, tmem);
      else few_tile<16>(p, c, w, t, t.head, split, slice, b0, n, tmem);
    } else {
      tile(p, c, w, t, t.head, split, slice, b0, n, tmem, 0);
    }
  }
  // tile i of a walk, -1: there is none
  __device__ __forceinline__ static AttnTile tile_at(const TileCtx &c, const Window &w, const AttnTile *tile_slot, int i) {
    AttnTile t;
    t.found = -1;
    // (tile 0 was there before c.sync)
    if (i == 0 || warp_wait(w.tile_bar + 8 * (i & 1), ((i - 1) >> 1) & 1, c.status, ATTN_WAIT_TILE_TIMEOUT)) t = tile_slot[i & 1];
    return t;
  }

  __device__ __forceinline__ static void run(const Params &p, const TileCtx &c) {
    const int warp = c.tid >> 5, lane = c.tid & 31;
    const int split = WALK ? 1 : p.split, stages = p.stages;
    const int slice = c.block_x() & (split - 1);   // (split: a power of two)
    const Window w = window(p, smem_u32(c.smem));
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(c.smem + 8 * kBars);
    AttnTile *tile_slot = reinterpret_cast<AttnTile *>(c.smem + 512);   // (two, in a walk)

    if (warp == kIssuer && !c.tmem_given) {
      tmem_alloc(smem_u32(tmem_slot), p.tmem_cols);
      if (!c.persistent) tmem_relinquish();
    }
    int loaded = 0;
    if (warp == kProducer) {
      // all of this needs no memory: it runs while the previous kernel ends
      if (lane < stages) {
        mbar_init(w.full0 + 8 * lane, 1);
        mbar_init(w.empty0 + 8 * lane, 1);
      }
      static_assert(kBars - 2 * kAttnMaxStages <= 32 && 8 * kBars + 4 <= 512 && 2 * sizeof(AttnTile) <= 256, "one lane a barrier, and the header's room");
      if (lane < kBars - 2 * kAttnMaxStages) mbar_init(w.q_bar + 8 * lane, arrivals(w, lane));
      if (lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &p.map_q : lane == 1 ? &p.map_k : &p.map_v) : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      if (lane == 0) {
        tile_slot->head = c.block_x() >> log2_of(split);
        tile_slot->loads = tile_slot->queries = 0;
        for (int x = 0; x < 2; ++x) tile_slot->blocks[x] = tile_slot->outs[x] = 0;
      }
      c.dependency_wait();
      find_tile(p, c.block_y(), c.gy, lane, tile_slot, c.status);
      const AttnTile t = *tile_slot;
      const bool few = t.found && few_rows(p, t);
      const int active = t.found ? (sub_tile(p, t, 0).npos * p.group + 31) >> 5 : 0;   // quarters of the (first) tile that hold a row
      int b0 = 0, n = 0;
      if (t.found) my_blocks(t, split, slice, b0, n);
      loaded = min(stages, 2 * n);
      if (elect_one()) {
        if (split > 1 && t.found) {
          // what this CTA will receive: (m, l) of every row from every rank, and the columns (few rows: dims) that it owns
          if (few) {
            const int r = t.npos * p.group <= 8 ? 8 : kAttnFewRows;
            mbar_expect_tx(w.join_bar, (uint32_t)(split * r * 8 + w.chunks * 64 * r * 4));
          } else {
            int owned = 0;
            for (int ch = slice; ch < w.chunks * 4; ch += split) ++owned;
            mbar_expect_tx(w.stats_bar, (uint32_t)(split * active * 32 * 8));
            if (owned) mbar_expect_tx(w.join_bar, (uint32_t)(owned * split * active * 32 * 64));
          }
        }
        if (n > 0) {   // the first round of the ring: every slot is free
          load_q(p, w, t);
          for (int i = 0; i < loaded; ++i) load(p, w, t, b0, i, (uint32_t)i);
        }
      }
      __syncwarp();
    } else {
      c.dependency_wait();
    }
    tc_fence_before();
    c.sync();
    tc_fence_after();
    // this CTA's barriers are up: its peers may push (they wait for that only when they have something to push)
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const uint32_t tmem = c.tmem_given ? c.tmem_base : *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    int b0, n;
    if constexpr (WALK) {
      if (warp == kProducer) {
        lead(p, c, w, tile_slot, loaded, lane);
      } else if (warp == kIssuer) {
#pragma unroll 1
        for (int i = 0;; ++i) {
          const AttnTile t = tile_at(c, w, tile_slot, i);
          if (t.found < 0) break;
          if (t.found) {
            my_blocks(t, 1, 0, b0, n);
            issue(p, c, w, t, b0, n, few_rows(p, t), tmem);
          }
          if (elect_one()) mbar_arrive(w.done_bar + 8 * (i & 1));
          __syncwarp();
        }
      } else {
#pragma unroll 1
        for (int i = 0;; ++i) {
          const AttnTile t = tile_at(c, w, tile_slot, i);
          if (t.found < 0) break;
          if (t.found) {
            my_blocks(t, 1, 0, b0, n);
            rows(p, c, window(p, anew(w.full0)), t, 1, 0, b0, n, few_rows(p, t), anew(tmem));
          }
          __syncwarp();
          fence_async_smem();   // what this thread wrote over the queries comes before the next ones
          tc_fence_before();
          mbar_arrive(w.done_bar + 8 * (i & 1));
        }
      }
    } else {
      const AttnTile t = *tile_slot;
      if (t.found) {   // (the same for every CTA of a cluster)
        my_blocks(t, split, slice, b0, n);
        const bool few = few_rows(p, t);
        if (warp == kProducer) {
          if (n > 0 && elect_one()) load_run(p, c, w, t, b0, loaded, 2 * n);
          __syncwarp();
        } else if (warp == kIssuer) {
          issue(p, c, w, t, b0, n, few, tmem);
        }
        rows(p, c, w, t, split, slice, b0, n, few, tmem);
      } else if (split > 1) {
        cluster_wait();
      }
    }
    __syncwarp();
    tc_fence_before();
    c.sync();
    if (warp == kIssuer && !c.tmem_given) tmem_dealloc(tmem, p.tmem_cols);
    if (c.persistent && c.tid < kBars) {   // the next tile of a persistent CTA initialises them again
      const int s = c.tid < kAttnMaxStages ? c.tid : c.tid - kAttnMaxStages;
      if (c.tid >= 2 * kAttnMaxStages || s < stages) mbar_inval(w.full0 + 8 * c.tid);
    }
  }

  // V as an operand whose rows are keys ("MN-major"): its 64-column chunks lie `chunk_step` bytes apart (leading offset),
  // groups of 8 keys 1024 bytes (stride offset), 16 keys -- one instruction -- 2048
  __device__ __forceinline__ static uint32_t v_desc(uint32_t addr, uint32_t chunk_step) { return ((addr >> 4) & 0x3fffu) | ((chunk_step >> 4) << 16); }
  __device__ __forceinline__ static uint32_t k_major_desc(uint32_t addr) { return ((addr >> 4) & 0x3fffu) | (1u << 16); }

  __device__ __forceinline__ static void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

  // In a walk the compiler would compute all that follows from x once, before the first tile, and hold it in registers that a row's
  // scores need (396 bytes of spills, prompts a fifth slower): x is another one for every tile.
  template <class V>
  __device__ __forceinline__ static V anew(V x) {
    if (WALK) asm volatile("" : "+r"(x));
    return x;
  }

  // ---- whole tiles: rows in the lanes ----

  // A slot of the ring and the phase its barrier is in, carried along: loads are `step` apart (divisions would idle the tensor pipe).
  struct RingAt {
    uint32_t slot, phase;
    __device__ __forceinline__ void advance(uint32_t step, uint32_t stages) {   // step <= stages
      slot += step;
      if (slot >= stages) slot -= stages, phase ^= 1;
    }
  };
  __device__ __forceinline__ static RingAt ring_at(const AttnTile &t, uint32_t load, uint32_t stages) {   // load 0 or 1 of the tile
    return WALK ? RingAt{(t.loads + load) % stages, (t.loads + load) / stages & 1u} : RingAt{load, 0};
  }

  // S = Q K^T of tile x and the block of keys at k; `wait`: nobody has waited for them yet, `last`: no other tile reads them after it
  __device__ __forceinline__ static bool scores(const Params &p, const TileCtx &c, const Window &w, const RingAt &k, uint32_t tmem, int x, bool wait, bool last) {
    const uint32_t idesc = umma_idesc(1, kAttnKeys), q_lo = k_major_desc(w.q + x * w.tile_bytes);
    const int ksteps = (p.dim + 15) >> 4;   // 16 dims a step (the TMA filled up what dim does not have)
    if (wait) {
      if (!mbar_wait(w.full0 + 8 * k.slot, k.phase, c.status, ATTN_WAIT_KV_TIMEOUT)) return false;
      tc_fence_after();
    }
    const uint32_t k_lo = k_major_desc(w.ring + k.slot * w.tile_bytes);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t off = (uint32_t)(i >> 2) * (kAttnChunkBytes >> 4) + 2 * (i & 3);
      if (i < ksteps) umma_ss<1>(tmem + 256u * x, q_lo + off, k_lo + off, idesc, i > 0);
    }
    if (last) umma_commit(w.empty0 + 8 * k.slot);
    umma_commit(w.s_bar + 8 * x);
    return true;
  }

  // The MMAs run in the order they are issued, and two tiles take turns, one's MMAs under the other's exponentials.
  // Where p has columns of its own (p_col), S of block j + 1 is made as soon as the threads have S of block j in their
  // registers; else p lies over S, and it follows p V of block j.  p V starts with the 64 keys whose p comes first.
  // (Blocks as two halves of 64 keys that go round by themselves are no faster: prompts this long run at the power limit.)
  __device__ __forceinline__ static bool multiply(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int n, uint32_t tmem) {
    const uint32_t idesc = umma_idesc(1, w.chunks * 64) | (1u << 16), stages = (uint32_t)p.stages;
    int nx[2] = {n, 0};
    if (T == 2) nx[0] = sub_blocks(sub_tile(p, t, 0), n), nx[1] = sub_blocks(sub_tile(p, t, 1), n);
    RingAt k = ring_at(t, 0, stages), v = ring_at(t, 1, stages);
    const uint32_t g[2] = {blocks(t, 0), T == 2 ? blocks(t, 1) : 0u};
    // block j is read by tile 0, if that has so many, and then by tile 1: the first waits for it, the last gives it up
    auto first = [&](int j, int x) { return T == 1 || x == 0 || j >= nx[0]; };
    auto last = [&](int j, int x) { return T == 1 || x == 1 || j >= nx[1]; };
    for (int x = 0; x < T; ++x)
      if (nx[x] > 0 && !scores(p, c, w, k, tmem, x, first(0, x), last(0, x))) return false;
    k.advance(2, stages);
    for (int j = 0; j < n; ++j) {
      const uint32_t v_lo = v_desc(w.ring + v.slot * w.tile_bytes, kAttnChunkBytes);
#pragma unroll
      for (int x = 0; x < T; ++x) {
        if (T == 2 && j >= nx[x]) continue;
        const bool more = j + 1 < nx[x];
        if (p.p_col && more) {
          if (!mbar_wait(w.c_bar + 8 * x, (g[x] + j) & 1, c.status, ATTN_WAIT_PROBS_TIMEOUT)) return false;
          tc_fence_after();
          if (!scores(p, c, w, k, tmem, x, first(j + 1, x), last(j + 1, x))) return false;
        }
        if (first(j, x) && !mbar_wait(w.full0 + 8 * v.slot, v.phase, c.status, ATTN_WAIT_KV_TIMEOUT)) return false;
        const uint32_t pt = tmem + 256u * x + (uint32_t)p.p_col;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!mbar_wait(w.p_bar + 16 * x + 8 * half, (g[x] + j) & 1, c.status, ATTN_WAIT_PROBS_TIMEOUT)) return false;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t step = (uint32_t)(4 * half + i);   // of 16 keys
            umma_ts_bf16(tmem + 256u * x + 128, pt + 8 * step, v_lo + 128 * step, idesc, j > 0 || half + i > 0);
          }
        }
        if (last(j, x)) umma_commit(w.empty0 + 8 * v.slot);
        if (p.p_col) umma_commit(w.pv_bar + 8 * x);
        else if (more && !scores(p, c, w, k, tmem, x, first(j + 1, x), last(j + 1, x))) return false;
        if (T == 2 && !more) umma_commit(w.o_bar + 8 * x);
      }
      v.advance(2, stages);
      k.advance(2, stages);
    }
    return true;
  }

  // (a whole warp gives up or goes on: what follows are warp-wide tensor-memory instructions)
  __device__ __forceinline__ static bool warp_wait(uint32_t bar, uint32_t parity, int *status, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
  }

  // Values past the end of the sequence are the next one's, or whatever the buffer holds: p is 0 there, but 0 * NaN is not,
  // so those rows of V become zeros.  `first` of `threads` threads; the block's V is load 2 j + 1 of the ring.
  __device__ __forceinline__ static bool clear_tail(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int j, int have, int first, int threads) {
    const uint32_t i = loads(t) + 2u * j + 1u, s = i % (uint32_t)p.stages;
    const bool ok = warp_wait(w.full0 + 8 * s, (i / (uint32_t)p.stages) & 1, c.status, ATTN_WAIT_KV_TIMEOUT);
    const uint32_t v = w.ring + s * w.tile_bytes;
    if (ok)
      for (int ch = 0; ch < w.chunks; ++ch)
        for (int k = first; k < (kAttnKeys - have) * 8; k += threads) st_shared_u4(v + ch * kAttnChunkBytes + have * 128 + k * 16, 0, 0, 0, 0);
    fence_async_smem();
    return ok;
  }

  // the largest of three
  __device__ __forceinline__ static float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
  }
  // columns behind `seen` of a row's scores do not count
  template <int G>
  __device__ __forceinline__ static void mask(uint32_t (&r)[G][32], int seen) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (32 * g + i > seen) r[g][i] = __float_as_uint(-INFINITY);
  }
  // The values of a tcgen05.ld that has been waited for: no use of them may move before the wait
  __device__ __forceinline__ static void loaded_scores(uint32_t (&r)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
  }
  // The scores of a row: the largest of G x 32 (with m), then 32 of their exponentials as bf16 into tensor memory
  template <bool MASKED, int G>
  __device__ __forceinline__ static float largest(uint32_t (&r)[G][32], int seen, float m) {
    float mx[4] = {m, m, m, m};
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        if (MASKED && 32 * g + i > seen) r[g][i] = __float_as_uint(-INFINITY);
        if (MASKED && 32 * g + i + 1 > seen) r[g][i + 1] = __float_as_uint(-INFINITY);
        mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(r[g][i]), __uint_as_float(r[g][i + 1]));
      }
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  }
  __device__ __forceinline__ static void exponentials(uint32_t p_tmem, const uint32_t (&r)[32], float sc, float mc, float2 (&sum)[2]) {
    const float2 sc2 = make_float2(sc, sc), mc2 = make_float2(-mc, -mc);
    uint32_t q[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 a = fma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), sc2, mc2);
      a.x = exp2_approx(a.x), a.y = exp2_approx(a.y);
      sum[i & 1] = add2(sum[i & 1], a);   // (two chains: one alone is 64 adds deep, and cost a tenth of a block of 64 dims)
      q[i] = f2_to_bf16x2(a.x, a.y);   // the second product takes bf16: half a step of p, as of the output
    }
    tmem_st_32x16(p_tmem, q);
  }

  __device__ __forceinline__ static void tile(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int head, int split, int slice,
                                              int b0, int n, uint32_t tmem_base, int x) {
    const uint32_t tmem = tmem_base + 256u * x;
    const int tid = anew(c.tid), warp = tid >> 5, lane = tid & 31;
    const int quad = (anew(threadIdx.x) >> 5) & 3;   // hardware warp w may only touch TMEM lanes [32 * (w % 4), +32)
    const int rows = t.npos * p.group, row = quad * 32 + lane, active = (rows + 31) >> 5;
    const bool mine = warp < kProducer && quad < active;   // this warp owns rows (the others only keep the barriers going)
    const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
    float m = -INFINITY, l = 0.f;   // the maximum the exponentials are taken against, and their sum
    bool ok = true;
    const uint32_t before = blocks(t, x);
    const uint32_t s_bar = w.s_bar + 8 * x, p_bar = w.p_bar + 16 * x, pv_bar = w.pv_bar + 8 * x, c_bar = w.c_bar + 8 * x;
    if (!mine && warp < kProducer) {
      for (int j = 0; j < n && ok; ++j) {
        ok = warp_wait(s_bar, (before + j) & 1, c.status, ATTN_WAIT_SCORES_TIMEOUT);
        if (p.p_col) mbar_arrive(c_bar);
        if (p.p_col && j > 0 && ok) ok = warp_wait(pv_bar, (before + j - 1) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
        mbar_arrive(p_bar);
        mbar_arrive(p_bar + 8);
      }
    }
    if (mine && n > 0) {
      const int limit = row < rows ? (p.causal ? min(t.last0 + row / p.group, t.kv_len - 1) : t.kv_len - 1) : -1;   // last key this row sees
      const float sc = p.scale_log2;
#pragma unroll 1
      for (int j = 0; j < n && ok; ++j) {
        const int key0 = (b0 + j) * kAttnKeys;
        ok = warp_wait(s_bar, (before + j) & 1, c.status, ATTN_WAIT_SCORES_TIMEOUT);
        if (!ok) break;
        tc_fence_after();
        const int seen = limit - key0;   // columns 0..seen of this block count
        const bool masked = __any_sync(0xffffffffu, seen < kAttnKeys - 1);
        // A row's 128 scores at once; in a walk, which leaves fewer registers, the second 64 twice, for the maximum and for their
        // exponentials (with all at once 276 bytes of spills: 60 prompts of 256 tokens 49 us, so 44; without a walk 57 and 58).
        constexpr int G = WALK ? 2 : 4;
        uint32_t r[G][32];
        float mx = m;
#pragma unroll
        for (int col = kAttnKeys - 32 * G; col >= 0; col -= 32 * G) {
#pragma unroll
          for (int g = 0; g < G; ++g) tmem_ld_32x32(trow + col + 32 * g, r[g]);
          tmem_ld_wait();
          if (!WALK && p.p_col) {
            tc_fence_before();
            mbar_arrive(c_bar);   // S may be overwritten
          }
          if (WALK)
#pragma unroll
            for (int g = 0; g < G; ++g) loaded_scores(r[g]);
          mx = masked ? largest<true>(r, seen - col, mx) : largest<false>(r, seen - col, mx);
        }
        if (p.p_col && j > 0) {   // p's columns are free, and O is whole, once p V of block j - 1 is done
          ok = warp_wait(pv_bar, (before + j - 1) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
          tc_fence_after();
        }
        // O follows a larger maximum only when that grew by more than 2^8: p stays below 2^8 and the sums in fp32 lose
        // nothing, and O mostly stays where it is.  (Without p_col s_bar stands for every MMA before it: block j - 1 is in O.)
        if (__any_sync(0xffffffffu, (mx - m) * sc > 8.f)) {
          const float f = mx == -INFINITY ? 1.f : exp2_approx((m - mx) * sc);
          m = mx;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int col = 0; col < w.chunks * 64; col += 16) {
              uint32_t o[16];
              tmem_ld_32x16(trow + 128 + col, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st_32x16(trow + 128 + col, o);
            }
          }
        }
        const int have = t.kv_len - key0;
        if (have < kAttnKeys && ok) ok = clear_tail(p, c, w, t, j, have, row, active * 32);
        const float mc = m == -INFINITY ? 0.f : m * sc;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const uint32_t pt = trow + (uint32_t)p.p_col;   // (over S, p of the first 64 keys stays clear of the scores of the others)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          exponentials(pt + 16 * g, r[g & (G - 1)], sc, mc, sum);
          if (WALK && g < 2) tmem_ld_32x32(trow + 64 + 32 * g, r[g]);
          if (g & 1) {
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(p_bar + 8 * (g >> 1));
          }
          if (WALK && g == 1) {
            tmem_ld_wait();
            loaded_scores(r[0]);
            loaded_scores(r[1]);
            if (p.p_col) {
              tc_fence_before();
              mbar_arrive(c_bar);   // S may be overwritten
            }
            if (masked) mask(r, seen - 64);
          }
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (ok) ok = warp_wait(w.o_bar + 8 * x, outs(t, x) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
      tc_fence_after();
    }
    if (T == 1 && split > 1) {
      join(p, c, w, t, head, split, slice, n, rows, row, mine, ok, trow, m, l);
    } else if (mine && ok) {
      // Through the rows of the Q tile, which no MMA reads any more (swizzled as the TMA left them), so that a row's dims leave
      // as whole lines: thread by thread, 16 bytes of 32 rows at a time, the stores took 2600 clocks of 128 dims, so 600.
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const uint32_t stage = w.q + x * w.tile_bytes + (uint32_t)(quad * 32) * 128u;
#pragma unroll 1
      for (int col = 0; col < p.dim; col += 32) {
        uint32_t r[32];
        if (n > 0) {
          tmem_ld_32x32(trow + 128 + col, r);
          tmem_ld_wait();
        }
        const uint32_t line = stage + (uint32_t)(col >> 6) * kAttnChunkBytes + (uint32_t)lane * 128u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = l == 0.f ? 0.f : __uint_as_float(r[8 * i + k]) * inv;   // a row without keys: zeros
          st_shared_u4(line + (uint32_t)(((((col >> 3) & 7) + i) ^ (lane & 7)) << 4), f2_to_bf16x2(v[0], v[1]), f2_to_bf16x2(v[2], v[3]),
                       f2_to_bf16x2(v[4], v[5]), f2_to_bf16x2(v[6], v[7]));
        }
      }
      __syncwarp();
      const int per_row = p.dim >> 3, lanes = per_row <= 8 ? 8 : 16, sub = lane & (lanes - 1);   // 16-byte pieces of a row; lanes that share one
      const int i0 = lanes == 8 ? lane >> 3 : lane >> 4, step = 32 / lanes;
      int g = quad * 32 + i0, pos = g / p.group;   // of the first row: head of the group, position
      g -= pos * p.group;
      uint16_t *out = p.out + ((size_t)(t.q0 + pos) * p.heads + head * p.group + g) * p.dim + 8 * sub;
      const size_t next = (size_t)(p.heads - p.group) * p.dim;   // from the group's heads to those of the next position
#pragma unroll 4
      for (int i = i0; i < 32; i += step) {
        if (sub < per_row && quad * 32 + i < rows)
          *reinterpret_cast<float4 *>(out) = ld_shared_f4(stage + (uint32_t)(sub >> 3) * kAttnChunkBytes + (uint32_t)i * 128u + (uint32_t)(((sub & 7) ^ (i & 7)) << 4));
        out += step * p.dim;
        for (g += step; g >= p.group; g -= p.group) out += next;
      }
    }
  }

  // The slices of a tile become one result (all threads of every CTA of the cluster).
  __device__ __forceinline__ static void join(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int head, int split, int slice, int n,
                                              int rows, int row, bool mine, bool ok, uint32_t trow, float m, float l) {
    cluster_wait();
    cluster_sync_all();   // every rank's MMAs are done: Q and the ring are free everywhere
    if (!mine) return;
    const float mlog = m * p.scale_log2;   // in powers of two
    const uint32_t area = w.q, recv = area + (uint32_t)(split * kAttnRows * 8);
    for (int r = 0; r < split; ++r)
      st_async_f2(peer_smem(area + (uint32_t)(slice * kAttnRows + row) * 8, r), peer_smem(w.stats_bar, r), mlog, l);
    if (!warp_wait(w.stats_bar, 0, c.status, ATTN_WAIT_PEERS_TIMEOUT)) ok = false;
    float top = -INFINITY, sum = 0.f;
    for (int r = 0; r < split; ++r) top = fmaxf(top, ld_shared_f2(area + (uint32_t)(r * kAttnRows + row) * 8).x);
    if (top == -INFINITY) top = 0.f;
    for (int r = 0; r < split; ++r) {
      const float2 s = ld_shared_f2(area + (uint32_t)(r * kAttnRows + row) * 8);
      sum += s.y * exp2_approx(s.x - top);
    }
    const float f = l == 0.f ? 0.f : exp2_approx(mlog - top) / sum;
    const int pieces = w.chunks * 4;   // of 16 columns
#pragma unroll 1
    for (int ch = 0; ch < pieces; ++ch) {
      uint32_t r[16];
      if (n > 0) {
        tmem_ld_32x16(trow + 128 + ch * 16, r);
        tmem_ld_wait();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(r[i]) * f);
      const uint32_t slot = recv + (uint32_t)((ch / split) * split + slice) * (16 * kAttnRows * 4);
      const uint32_t dst = peer_smem(slot + (uint32_t)row * 16, ch % split), bar = peer_smem(w.join_bar, ch % split);
#pragma unroll
      for (int i = 0; i < 4; ++i) st_async_u4(dst + (uint32_t)(i * kAttnRows * 16), bar, r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    }
    if (slice >= pieces) return;   // owns no columns
    if (!warp_wait(w.join_bar, 0, c.status, ATTN_WAIT_PEERS_TIMEOUT) || !ok || row >= rows) return;
    uint16_t *out = out_row(p, t, head, row);
#pragma unroll 1
    for (int ch = slice; ch < pieces; ch += split) {
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = 0.f;
      for (int r = 0; r < split; ++r) {   // rank order: the sum is deterministic
        const uint32_t src = recv + (uint32_t)((ch / split) * split + r) * (16 * kAttnRows * 4) + (uint32_t)row * 16;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 a = ld_shared_f4(src + (uint32_t)(k * kAttnRows * 16));
          v[4 * k] += a.x, v[4 * k + 1] += a.y, v[4 * k + 2] += a.z, v[4 * k + 3] += a.w;
        }
      }
      store16(out, ch * 16, p.dim, v);
    }
  }

  // ---- tiles of few rows: keys, then dims, in the lanes ----

  // p^T of a block: 16 rows x 128 keys bf16, K-major in two 64-key chunks; two of them lie over the rows of the Q tile that a
  // tile of few rows does not have
  __device__ __forceinline__ static uint32_t pt_smem(const Window &w, uint32_t j) { return w.q + 2048u + (j & 1) * 4096u; }

  // S^T of block j + 1 = K Q^T goes into the other of two buffers while the threads work on block j (block j - 1 is done with
  // it), then O^T += V^T p^T of block j.  The ring's loads are used in the order K0 K1 V0 K2 V1 ...
  __device__ __forceinline__ static bool multiply_few(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int n, uint32_t tmem) {
    const uint32_t idesc_s = umma_idesc(1, kAttnFewRows), idesc_o = idesc_s | (1u << 15), stages = (uint32_t)p.stages;   // V transposed
    const uint32_t q_lo = k_major_desc(w.q), chunk_step = w.chunks == 2 ? kAttnChunkBytes : 0;   // (a head of one chunk fills 64 lanes, the others get it again)
    const int ksteps = (p.dim + 15) >> 4;
    RingAt k = ring_at(t, 0, stages), v = ring_at(t, 1, stages);
    for (int j = -1; j < n; ++j) {
      const uint32_t g = blocks(t, 1) + (uint32_t)j;
      if (j + 1 < n) {
        if (!mbar_wait(w.full0 + 8 * k.slot, k.phase, c.status, ATTN_WAIT_KV_TIMEOUT)) return false;
        tc_fence_after();
        const uint32_t k_lo = k_major_desc(w.ring + k.slot * w.tile_bytes);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t off = (uint32_t)(i >> 2) * (kAttnChunkBytes >> 4) + 2 * (i & 3);
          if (i < ksteps) umma_ss<1>(tmem + ((g + 1) & 1) * kAttnFewRows, k_lo + off, q_lo + off, idesc_s, i > 0);
        }
        umma_commit(w.empty0 + 8 * k.slot);
        umma_commit(w.sf_bar + 8 * ((g + 1) & 1));
        k.advance(2, stages);
      }
      if (j < 0) continue;
      // (the next block's p may be there before this wait is: a barrier for each of the two)
      if (!mbar_wait(w.full0 + 8 * v.slot, v.phase, c.status, ATTN_WAIT_KV_TIMEOUT) ||
          !mbar_wait(w.pf_bar + 8 * (g & 1), (g >> 1) & 1, c.status, ATTN_WAIT_PROBS_TIMEOUT))
        return false;
      tc_fence_after();
      const uint32_t v_lo = v_desc(w.ring + v.slot * w.tile_bytes, chunk_step), pt_lo = k_major_desc(pt_smem(w, g));
#pragma unroll
      for (int i = 0; i < kAttnKeys / 16; ++i)
        umma_ss<1>(tmem + 128, v_lo + 128 * i, pt_lo + (uint32_t)(i >> 2) * 128 + 2 * (i & 3), idesc_o, j > 0 || i > 0);
      umma_commit(w.empty0 + 8 * v.slot);
      umma_commit(w.pvf_bar);
      v.advance(2, stages);
    }
    return true;
  }

  // the four warps that own the lanes (barrier 9 or 10)
  __device__ __forceinline__ static void quads_sync(const TileCtx &c) { asm volatile("bar.sync %0, 128;" ::"r"(c.bar_id + 8) : "memory"); }
  __device__ __forceinline__ static bool quads_any(const TileCtx &c, bool x) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)x), "r"(c.bar_id + 8)
        : "memory");
    return any != 0;
  }
  // over the 128 lanes, for each of R values; everyone gets it
  template <class Op, int R>
  __device__ __forceinline__ static void quads_reduce(const TileCtx &c, const Window &w, int quad, int lane, float (&v)[R]) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = Op::apply(v[i], __shfl_xor_sync(0xffffffffu, v[i], off));
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < R / 4; ++i)
        st_shared_u4(w.xch + (uint32_t)(quad * 64 + i * 16), __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                     __float_as_uint(v[4 * i + 3]));
    quads_sync(c);
#pragma unroll
    for (int i = 0; i < R / 4; ++i) {
      float4 a = ld_shared_f4(w.xch + (uint32_t)(i * 16));
#pragma unroll
      for (int k = 1; k < 4; ++k) {
        const float4 b = ld_shared_f4(w.xch + (uint32_t)(k * 64 + i * 16));
        a.x = Op::apply(a.x, b.x), a.y = Op::apply(a.y, b.y), a.z = Op::apply(a.z, b.z), a.w = Op::apply(a.w, b.w);
      }
      v[4 * i] = a.x, v[4 * i + 1] = a.y, v[4 * i + 2] = a.z, v[4 * i + 3] = a.w;
    }
  }
  template <int R>
  __device__ __forceinline__ static void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[R]) {
    if constexpr (R == 16) tmem_ld_32x16(taddr, r);
    else
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                   : "r"(taddr));
    tmem_ld_wait();
  }
  template <int R>
  __device__ __forceinline__ static void tmem_st_rows(uint32_t taddr, const uint32_t (&r)[R]) {
    if constexpr (R == 16) tmem_st_32x16(taddr, r);
    else
      asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                   "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                   : "memory");
    tmem_st_wait();
  }

  template <int R>   // rows worked on: 8 or 16
  __device__ __forceinline__ static void few_tile(const Params &p, const TileCtx &c, const Window &w, const AttnTile &t, int head, int split, int slice,
                                                  int b0, int n, uint32_t tmem) {
    const int tid = anew(c.tid), warp = tid >> 5, lane = tid & 31, quad = (anew(threadIdx.x) >> 5) & 3, at = quad * 32 + lane;   // key of the block, then dim
    const bool mine = warp < 4;
    const int rows = t.npos * p.group;
    const uint32_t tlane = tmem + ((uint32_t)(quad * 32) << 16);
    float m[R], l[R];   // of every row: the maximum (in powers of two) the exponentials are taken against, the same in all lanes; this key's part of the sum
    bool ok = true;
#pragma unroll
    for (int i = 0; i < R; ++i) m[i] = -INFINITY, l[i] = 0.f;
    if (mine && n > 0) {
      const float sc = p.scale_log2;
      const int last = p.causal ? min(t.last0, t.kv_len - 1) : t.kv_len - 1;   // of the first position: every row sees up to here
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const int key0 = (b0 + j) * kAttnKeys, key = key0 + at;
        const uint32_t g = blocks(t, 1) + (uint32_t)j;
        if (ok) ok = warp_wait(w.sf_bar + 8 * (g & 1), (g >> 1) & 1, c.status, ATTN_WAIT_SCORES_TIMEOUT);   // (these four warps meet in every block: they go on together after a wait that gave up)
        tc_fence_after();
        uint32_t r[R];
        tmem_ld_rows<R>(tlane + (g & 1) * kAttnFewRows, r);
        float s[R];
        bool grown = false;
#pragma unroll
        for (int i = 0; i < R; ++i) s[i] = i < rows ? __uint_as_float(r[i]) * sc : -INFINITY;
        if (key0 + kAttnKeys - 1 > last) {   // not every row sees the whole block
          int limit = last, left = p.group;
#pragma unroll
          for (int i = 0; i < R; ++i) {
            if (key > limit) s[i] = -INFINITY;
            if (--left == 0) left = p.group, limit = p.causal ? min(limit + 1, t.kv_len - 1) : limit;
          }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) grown |= s[i] > m[i] + 8.f;
        if (quads_any(c, grown)) {   // some row's maximum grew by more than 2^8 (or is the first): as in tile()
          float mx[R];
#pragma unroll
          for (int i = 0; i < R; ++i) mx[i] = fmaxf(m[i], s[i]);
          quads_reduce<OpMax, R>(c, w, quad, lane, mx);
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float f = mx[i] == -INFINITY ? 1.f : exp2_approx(m[i] - mx[i]);
            m[i] = mx[i];
            l[i] *= f;
            mx[i] = f;
          }
          if (j > 0) {   // block j - 1 has to be in O
            if (ok) ok = warp_wait(w.pvf_bar, (g - 1) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
            tc_fence_after();
            uint32_t o[R];
            tmem_ld_rows<R>(tlane + 128, o);
#pragma unroll
            for (int i = 0; i < R; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * mx[i]);
            tmem_st_rows<R>(tlane + 128, o);
          }
        }
        // (S of this block stands for block j - 2's products, which read this buffer: it was issued after them)
        const uint32_t pt = pt_smem(w, g) + (uint32_t)(at >> 6) * 2048u + (uint32_t)(at & 7) * 2u;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float e = exp2_approx(s[i] - (m[i] == -INFINITY ? 0.f : m[i]));
          l[i] += e;
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(pt + (uint32_t)(i * 128 + ((((at & 63) >> 3) ^ (i & 7)) << 4))), "h"(__bfloat16_as_ushort(__float2bfloat16_rn(e)))
                       : "memory");
        }
        const int have = t.kv_len - key0;
        if (have < kAttnKeys) {
          // (these threads may be a block ahead: V's barrier says which block it holds only once block j - 1 is through)
          if (j > 0 && ok) ok = warp_wait(w.pvf_bar, (g - 1) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
          if (ok) ok = clear_tail(p, c, w, t, j, have, at, 128);
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(w.pf_bar + 8 * (g & 1));
      }
      if (ok) ok = warp_wait(w.o_bar, outs(t, 0) & 1, c.status, ATTN_WAIT_OUT_TIMEOUT);
      tc_fence_after();
      quads_reduce<OpSum, R>(c, w, quad, lane, l);
    }
    uint32_t o[R];
    auto read_o = [&] {
#pragma unroll
      for (int i = 0; i < R; ++i) o[i] = 0u;
      if (n > 0) tmem_ld_rows<R>(tlane + 128, o);
    };
    if (split == 1) {
      if (!mine || !ok) return;
      read_o();
      if (at < p.dim)
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (i < rows) reinterpret_cast<__nv_bfloat16 *>(out_row(p, t, head, i))[at] = __float2bfloat16_rn(l[i] == 0.f ? 0.f : __uint_as_float(o[i]) / l[i]);
      return;
    }
    // The slices become one: rank r owns the dims [r * per, (r + 1) * per).  Everyone pushes (m, l) of its rows to all and its
    // part of O, as it is, to the owners, into memory kept for that; the owner weighs the parts.
    cluster_wait();
    if (!mine) return;
    const int dims = w.chunks * 64, per_log2 = log2_of(dims) - log2_of(split), per = 1 << per_log2;
    const uint32_t stats = w.few_join, recv = stats + kAttnFewStats;
    read_o();
    if (at < dims) {
      const int owner = at >> per_log2;
      const uint32_t dst = peer_smem(recv + (uint32_t)(slice * per + at - owner * per) * (R * 4), owner), bar = peer_smem(w.join_bar, owner);
#pragma unroll
      for (int i = 0; i < R / 4; ++i) st_async_u4(dst + 16 * i, bar, o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)   // lane r of quarter i % 4 tells rank r of row i
      if (quad == (i & 3) && lane < split) st_async_f2(peer_smem(stats + (uint32_t)(slice * R + i) * 8, lane), peer_smem(w.join_bar, lane), m[i], l[i]);
    __syncwarp();
    if (!warp_wait(w.join_bar, 0, c.status, ATTN_WAIT_PEERS_TIMEOUT)) ok = false;
    if (at < R) {   // what the ranks' parts of row `at` count
      float top = -INFINITY, sum = 0.f;
      for (int r = 0; r < split; ++r) top = fmaxf(top, ld_shared_f2(stats + (uint32_t)(r * R + at) * 8).x);
      if (top == -INFINITY) top = 0.f;
      for (int r = 0; r < split; ++r) {
        const float2 st = ld_shared_f2(stats + (uint32_t)(r * R + at) * 8);
        sum += st.y * exp2_approx(st.x - top);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      for (int r = 0; r < split; ++r) {
        const float2 st = ld_shared_f2(stats + (uint32_t)(r * R + at) * 8);
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(w.xch + (uint32_t)(r * R + at) * 4), "f"(st.y == 0.f ? 0.f : exp2_approx(st.x - top) * inv) : "memory");
      }
    }
    quads_sync(c);
    if (!ok) return;
    for (int i = at; i < per * rows; i += 128) {
      const int row = i >> per_log2, d = i & (per - 1);
      float v = 0.f;
      for (int r = 0; r < split; ++r) {   // rank order: the sum is deterministic
        const float f = ld_shared_f32(w.xch + (uint32_t)(r * R + row) * 4);
        if (f != 0.f) v = fmaf(f, ld_shared_f32(recv + (uint32_t)((r * per + d) * R + row) * 4), v);
      }
      if (slice * per + d < p.dim) reinterpret_cast<__nv_bfloat16 *>(out_row(p, t, head, row))[slice * per + d] = __float2bfloat16_rn(v);
    }
  }
};

using AttentionBf16 = Attention<1, false>;
using AttentionBf16Walk = Attention<1, true>;
using AttentionBf16Two = Attention<2, false>;

}  // namespace bfuse
