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
// the rows (thread = row = lane of tensor memory), warp 4 issues the TMA loads, warp 5 the MMAs.
// GridDim = (slices * kv heads, tiles); the tiles are counted from the sequence offsets on the device
// (`find_tile`), the host knows only their number at most: (total_q + seqs (P - 1)) / P.  The last
// tile of a sequence, the one with the most keys under a causal mask, comes first.
//
// Few rows over many keys: the `slices` CTAs of a tile form a thread-block cluster, each takes a run of
// its 128-key blocks, and they join through distributed shared memory as the k-slices of the GEMM body
// do -- first every rank's (m, l) of every row, then its O scaled by 2^(m_rank - m) / l, summed in rank
// order by the rank that owns the columns (deterministic).
//
// Tensor memory: S in columns 0-127, the bf16 p over its first 64, O in columns 128 up: 256 columns, so
// two CTAs share an SM and one's MMAs run under the other's exponentials.
#pragma once

#include "ops_umma.cuh"

namespace bfuse {

constexpr int kAttnThreads = 192;
constexpr int kAttnRows = 128;     // query rows of a tile
constexpr int kAttnKeys = 128;     // keys of a block
constexpr int kAttnChunkBytes = 128 * 128;   // 128 rows x 64 bf16: what one TMA box holds
constexpr int kAttnTmemCols = 256;
constexpr int kAttnMaxStages = 8;

enum AttnStatus : int {
  ATTN_WAIT_Q_TIMEOUT = 0x301,
  ATTN_WAIT_KV_TIMEOUT = 0x302,
  ATTN_WAIT_SLOT_TIMEOUT = 0x303,
  ATTN_WAIT_SCORES_TIMEOUT = 0x304,
  ATTN_WAIT_PROBS_TIMEOUT = 0x305,
  ATTN_WAIT_OUT_TIMEOUT = 0x306,
  ATTN_WAIT_PEERS_TIMEOUT = 0x307,
  ATTN_BAD_OFFSETS = -1,   // BFUSE_STATUS_BAD_OFFSETS: sequence offsets that fall, or that leave the tensors: that sequence is left out
};

__host__ __device__ constexpr int attn_chunks(int dim) { return dim <= 64 ? 1 : 2; }   // 64-element chunks of a head
__host__ __device__ constexpr int attn_tile_bytes(int dim) { return attn_chunks(dim) * kAttnChunkBytes; }
__host__ __device__ constexpr int attn_smem_bytes(int dim, int stages) { return kUmmaHeaderBytes + (1 + stages) * attn_tile_bytes(dim); }
// what the slices of a tile exchange at the end: (m, l) per rank and row, and per 16 owned columns 8 KB of every rank
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
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  int found;      // 0: this block has no tile
  int q0, npos;   // first token, positions (<= P) of the tile
  int kv0, kv_len;
  int last0;      // causal: key index (within the sequence) that the tile's first position may see last
  int keys;       // keys that any row of the tile may see
};

struct AttentionBf16 {
  using Params = AttentionParams;
  static constexpr int kMaxThreads = kAttnThreads;
  static constexpr int kMinBlocks = 2;   // two CTAs an SM: 168 registers a thread
  static constexpr bool kMemoryBound = false;
  static constexpr bool kUsesTmem = true;

  // Tile number t of the batch: sequence i has ceil(len_i / P) of them.  One warp; 256 sequences a round, 8 a lane,
  // so that a batch of single tokens costs one trip to memory for its offsets and not one per 32 sequences.
  __device__ __forceinline__ static AttnTile find_tile(const Params &p, int t, int lane, int *status) {
    AttnTile tile;
    tile.found = 0;
    int before = 0;   // tiles of the sequences before this round's
    for (int base = 0; base < p.seqs; base += 256) {
      const int s0 = base + lane * 8;
      int cu[9], n[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 9; ++i) cu[i] = s0 + i <= p.seqs ? __ldg(p.cu_q + s0 + i) : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] = 0;
        if (s0 + i < p.seqs) {
          if (cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > p.total_q) atomicCAS(status, 0, (int)ATTN_BAD_OFFSETS);
          else n[i] = (cu[i + 1] - cu[i] + p.positions - 1) / p.positions;
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
        const bool here = t >= at && t < at + mine;
        if (here) {
          bool done = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (!done && t < at + n[i]) {
              done = true;
              const int qt = n[i] - 1 - (t - at);   // the last positions first
              const int kv_a = __ldg(p.cu_kv + s0 + i), kv_b = __ldg(p.cu_kv + s0 + i + 1);
              const int q_len = cu[i + 1] - cu[i];
              tile.found = kv_a >= 0 && kv_b >= kv_a && kv_b <= p.total_kv;
              if (!tile.found) atomicCAS(status, 0, (int)ATTN_BAD_OFFSETS);
              tile.q0 = cu[i] + qt * p.positions;
              tile.npos = min(p.positions, q_len - qt * p.positions);
              tile.kv0 = kv_a;
              tile.kv_len = kv_b - kv_a;
              tile.last0 = tile.kv_len - q_len + qt * p.positions;
              tile.keys = p.causal ? max(0, min(tile.kv_len, tile.last0 + tile.npos)) : tile.kv_len;
            }
            at += n[i];
          }
        }
        const unsigned who = __ballot_sync(0xffffffffu, here);
        const int src = __ffs(who) - 1;
        tile.found = __shfl_sync(0xffffffffu, tile.found, src);
        tile.q0 = __shfl_sync(0xffffffffu, tile.q0, src);
        tile.npos = __shfl_sync(0xffffffffu, tile.npos, src);
        tile.kv0 = __shfl_sync(0xffffffffu, tile.kv0, src);
        tile.kv_len = __shfl_sync(0xffffffffu, tile.kv_len, src);
        tile.last0 = __shfl_sync(0xffffffffu, tile.last0, src);
        tile.keys = __shfl_sync(0xffffffffu, tile.keys, src);
        return tile;
      }
      before += total;
    }
    return tile;
  }

  __device__ __forceinline__ static void load_kv(const CUtensorMap *map, uint32_t dst, uint32_t bar, int chunks, int head, int token) {
    mbar_expect_tx(bar, (uint32_t)chunks * kAttnChunkBytes);
    for (int ch = 0; ch < chunks; ++ch) tma_load_3d(dst + ch * kAttnChunkBytes, map, bar, ch * 64, head, token);
  }

  // 16 finished columns of a row
  __device__ __forceinline__ static void store16(uint16_t *row, int col, int dim, const float (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (col + 8 * j < dim)
        *reinterpret_cast<uint4 *>(row + col + 8 * j) = make_uint4(f2_to_bf16x2(v[8 * j], v[8 * j + 1]), f2_to_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                                                                   f2_to_bf16x2(v[8 * j + 4], v[8 * j + 5]), f2_to_bf16x2(v[8 * j + 6], v[8 * j + 7]));
  }

  __device__ __forceinline__ static void run(const Params &p, const TileCtx &c) {
    const int warp = c.tid >> 5, lane = c.tid & 31;
    const int quad = (threadIdx.x >> 5) & 3;   // hardware warp w may only touch TMEM lanes [32 * (w % 4), +32)
    const int split = p.split, stages = p.stages;
    const int bx = c.block_x(), slice = bx % split, head = bx / split;
    const int chunks = attn_chunks(p.dim), tile_bytes = chunks * kAttnChunkBytes;

    // window: [0, 1024) barriers, tensor-memory pointer and the tile; from kUmmaHeaderBytes on Q, then the ring of
    // `stages` K / V blocks in the order K0 V0 K1 V1 ...
    uint64_t *bars = reinterpret_cast<uint64_t *>(c.smem);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kAttnMaxStages, q_bar = empty0 + 8 * kAttnMaxStages;
    const uint32_t s_bar = q_bar + 8, p_bar = q_bar + 16, o_bar = q_bar + 24, stats_bar = q_bar + 32, join_bar = q_bar + 40;
    constexpr int kBars = 2 * kAttnMaxStages + 6;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(c.smem + 8 * kBars);
    AttnTile *tile_slot = reinterpret_cast<AttnTile *>(c.smem + 256);
    const uint32_t q_smem = smem_u32(c.smem) + kUmmaHeaderBytes, ring = q_smem + tile_bytes;

    if (warp == 5 && !c.tmem_given) {
      tmem_alloc(smem_u32(tmem_slot), kAttnTmemCols);
      if (!c.persistent) tmem_relinquish();
    }
    c.dependency_wait();
    if (warp == 4) {
      const AttnTile t = find_tile(p, c.block_y(), lane, c.status);
      const int active = t.found ? (t.npos * p.group + 31) >> 5 : 0;   // warps that own a row
      if (lane == 0) {
        *tile_slot = t;
        for (int i = 0; i < stages; ++i) {
          mbar_init(full0 + 8 * i, 1);
          mbar_init(empty0 + 8 * i, 1);
        }
        mbar_init(q_bar, 1);
        mbar_init(s_bar, 1);
        mbar_init(p_bar, active > 0 ? active * 32 : 1);
        mbar_init(o_bar, 1);
        mbar_init(stats_bar, 1);
        mbar_init(join_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (split > 1 && t.found) {
          // what this CTA will receive: (m, l) of every row from every rank, and the columns that it owns
          int owned = 0;
          for (int ch = slice; ch < chunks * 4; ch += split) ++owned;
          mbar_expect_tx(stats_bar, (uint32_t)(split * active * 32 * 8));
          if (owned) mbar_expect_tx(join_bar, (uint32_t)(owned * split * active * 32 * 64));
        }
      }
      __syncwarp();
    }
    tc_fence_before();
    c.sync();
    tc_fence_after();
    const uint32_t tmem = c.tmem_given ? c.tmem_base : *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    const AttnTile t = *tile_slot;
    if (t.found) {   // (the same for every CTA of a cluster)
      const int nblocks = (t.keys + kAttnKeys - 1) / kAttnKeys, per = (nblocks + split - 1) / split;
      const int b0 = min(nblocks, slice * per), n = min(nblocks, b0 + per) - b0;   // this slice's blocks of keys
      if (warp == 4) produce(p, c, t, head, b0, n, full0, empty0, q_bar, q_smem, ring, chunks);
      else if (warp == 5) multiply(p, c, n, tmem, full0, empty0, q_bar, s_bar, p_bar, o_bar, q_smem, ring, chunks);
      const int rows = t.npos * p.group, row = quad * 32 + lane;
      const bool mine = warp < 4 && quad * 32 < rows;   // this warp owns rows
      float m = -INFINITY, l = 0.f;   // of this thread's row: the maximum the exponentials are taken against, and their sum
      bool ok = true;
      const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
      const int pos = row / p.group;
      if (mine && n > 0) {
        const int limit = row < rows ? (p.causal ? min(t.last0 + pos, t.kv_len - 1) : t.kv_len - 1) : -1;   // last key this row sees
        ok = softmax(p, c, t, limit, b0, n, trow, full0, s_bar, p_bar, ring, chunks, m, l, active_threads(rows));
        ok = warp_wait(o_bar, 0, c.status, ATTN_WAIT_OUT_TIMEOUT) && ok;
        tc_fence_after();
      }
      uint16_t *out = p.out + ((size_t)(t.q0 + pos) * p.heads + head * p.group + (row - pos * p.group)) * p.dim;
      if (split > 1) {
        join(p, c, split, slice, n, chunks, rows, row, mine, ok, trow, q_smem, stats_bar, join_bar, m, l, out);
      } else if (mine && ok) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int col = 0; col < p.dim; col += 32) {
          uint32_t r[32];
          if (n > 0) {
            tmem_ld_32x32(trow + 128 + col, r);
            tmem_ld_wait();
          }
          if (row < rows) {
            float v[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = l == 0.f ? 0.f : __uint_as_float(r[16 * h + j]) * inv;   // a row without keys: zeros
              store16(out, col + 16 * h, p.dim, v);
            }
          }
        }
      }
    }
    __syncwarp();
    tc_fence_before();
    c.sync();
    if (warp == 5 && !c.tmem_given) tmem_dealloc(tmem, kAttnTmemCols);
    if (c.persistent && c.tid < kBars) {   // the next tile of a persistent CTA initialises them again
      const int s = c.tid < kAttnMaxStages ? c.tid : c.tid - kAttnMaxStages;
      if (c.tid >= 2 * kAttnMaxStages || s < stages) mbar_inval(full0 + 8 * c.tid);
    }
  }

  __device__ __forceinline__ static int active_threads(int rows) { return min(128, (rows + 31) & ~31); }

  __device__ __forceinline__ static void produce(const Params &p, const TileCtx &c, const AttnTile &t, int head, int b0, int n, uint32_t full0,
                                                 uint32_t empty0, uint32_t q_bar, uint32_t q_smem, uint32_t ring, int chunks) {
    if (n > 0 && elect_one()) {
      const int tile_bytes = chunks * kAttnChunkBytes;
      mbar_expect_tx(q_bar, (uint32_t)(chunks * p.group * p.positions * 128));
      for (int ch = 0; ch < chunks; ++ch) tma_load_3d(q_smem + ch * kAttnChunkBytes, &p.map_q, q_bar, ch * 64, head * p.group, t.q0);
      uint32_t s = 0, ph = 1;   // (a slot's first use waits for nothing: parity 1 of a fresh barrier)
      for (int i = 0; i < 2 * n; ++i) {
        if (!mbar_wait(empty0 + 8 * s, ph, c.status, ATTN_WAIT_SLOT_TIMEOUT)) break;
        load_kv(i & 1 ? &p.map_v : &p.map_k, ring + s * tile_bytes, full0 + 8 * s, chunks, head, t.kv0 + (b0 + (i >> 1)) * kAttnKeys);
        if (++s == (uint32_t)p.stages) s = 0, ph ^= 1;
      }
    }
    __syncwarp();
  }

  __device__ __forceinline__ static void multiply(const Params &p, const TileCtx &c, int n, uint32_t tmem, uint32_t full0, uint32_t empty0,
                                                  uint32_t q_bar, uint32_t s_bar, uint32_t p_bar, uint32_t o_bar, uint32_t q_smem, uint32_t ring,
                                                  int chunks) {
    if (n > 0 && elect_one()) {
      const uint32_t idesc_s = umma_idesc(1, kAttnKeys), idesc_o = umma_idesc(1, chunks * 64) | (1u << 16);   // V: keys are its rows ("MN-major")
      const uint32_t tile16 = (uint32_t)(chunks * kAttnChunkBytes) >> 4;
      const uint32_t q_lo = ((q_smem >> 4) & 0x3fffu) | (1u << 16), ring_lo = (ring >> 4) & 0x3fffu;
      const int ksteps = (p.dim + 15) >> 4;   // 16 dims a step (the TMA filled up what dim does not have)
      uint32_t s = 0, ph = 0;
      bool ok = mbar_wait(q_bar, 0, c.status, ATTN_WAIT_Q_TIMEOUT);
      for (int j = 0; j < n && ok; ++j) {
        // S = Q K^T.  It may overwrite the p of block j - 1: the MMAs of one CTA run in the order they are issued
        ok = mbar_wait(full0 + 8 * s, ph, c.status, ATTN_WAIT_KV_TIMEOUT);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_lo = (ring_lo + s * tile16) | (1u << 16);
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t off = (uint32_t)(k >> 2) * (kAttnChunkBytes >> 4) + 2 * (k & 3);
          umma_ss<1>(tmem, q_lo + off, k_lo + off, idesc_s, k > 0);
        }
        umma_commit(empty0 + 8 * s);
        umma_commit(s_bar);
        if (++s == (uint32_t)p.stages) s = 0, ph ^= 1;
        // O += p V
        ok = mbar_wait(p_bar, j & 1, c.status, ATTN_WAIT_PROBS_TIMEOUT) && mbar_wait(full0 + 8 * s, ph, c.status, ATTN_WAIT_KV_TIMEOUT);
        if (!ok) break;
        tc_fence_after();
        // 64-column chunks of V lie one box apart (leading offset), groups of 8 keys 1024 bytes (stride offset)
        const uint32_t v_lo = (ring_lo + s * tile16) | ((uint32_t)(kAttnChunkBytes >> 4) << 16);
#pragma unroll
        for (int k = 0; k < kAttnKeys / 16; ++k) umma_ts_bf16(tmem + 128, tmem + 8 * k, v_lo + 128 * k, idesc_o, j > 0 || k > 0);
        umma_commit(empty0 + 8 * s);
        if (++s == (uint32_t)p.stages) s = 0, ph ^= 1;
      }
      umma_commit(o_bar);
      // the slot releases of the last uses are asynchronous: none may be in flight when the barriers go
      const int uses = 2 * n;
      for (int i = max(0, uses - p.stages); i < uses && ok; ++i)
        ok = mbar_wait(empty0 + 8 * (i % p.stages), (i / p.stages) & 1, c.status, ATTN_WAIT_SLOT_TIMEOUT);
      if (ok) mbar_wait(o_bar, 0, c.status, ATTN_WAIT_OUT_TIMEOUT);
    }
    __syncwarp();
  }

  // (a whole warp gives up or goes on: what follows are warp-wide tensor-memory instructions)
  __device__ __forceinline__ static bool warp_wait(uint32_t bar, uint32_t parity, int *status, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
  }

  // The online softmax of one row over this slice's blocks.  False: a wait gave up.
  __device__ __forceinline__ static bool softmax(const Params &p, const TileCtx &c, const AttnTile &t, int limit, int b0, int n, uint32_t trow,
                                                 uint32_t full0, uint32_t s_bar, uint32_t p_bar, uint32_t ring, int chunks, float &m_out, float &l_out,
                                                 int threads) {
    const float sc = p.scale_log2;
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int key0 = (b0 + j) * kAttnKeys;
      if (!warp_wait(s_bar, j & 1, c.status, ATTN_WAIT_SCORES_TIMEOUT)) return false;
      tc_fence_after();
      const int seen = limit - key0;   // columns 0..seen of this block count
      const bool masked = __any_sync(0xffffffffu, seen < kAttnKeys - 1);
      float mx = m;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t r[32];
        tmem_ld_32x32(trow + 32 * h, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) mx = fmaxf(mx, (masked && 32 * h + i > seen) ? -INFINITY : __uint_as_float(r[i]));
      }
      // O follows a larger maximum only when that grew by more than 2^8: p stays below 2^8 and the sums in fp32 lose
      // nothing, and O mostly stays where it is.  (s_bar stands for every MMA before it, so block j - 1 is in O.)
      if (__any_sync(0xffffffffu, (mx - m) * sc > 8.f)) {
        const float f = mx == -INFINITY ? 1.f : ex2((m - mx) * sc);
        m = mx;
        l *= f;
        if (j > 0) {
#pragma unroll 1
          for (int col = 0; col < chunks * 64; col += 16) {
            uint32_t r[16];
            tmem_ld_32x16(trow + 128 + col, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
            tmem_st_32x16(trow + 128 + col, r);
          }
        }
      }
      const float mc = m == -INFINITY ? 0.f : m * sc;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t r[32], q[16];
        tmem_ld_32x32(trow + 32 * h, r);
        tmem_ld_wait();
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float a = __uint_as_float(r[2 * i]), b = __uint_as_float(r[2 * i + 1]);
          if (masked && 32 * h + 2 * i > seen) a = -INFINITY;
          if (masked && 32 * h + 2 * i + 1 > seen) b = -INFINITY;
          a = ex2(fmaf(a, sc, -mc)), b = ex2(fmaf(b, sc, -mc));
          sum += a + b;
          q[i] = f2_to_bf16x2(a, b);   // the second product takes bf16: half a step of p, as of the output
        }
        l += sum;
        tmem_st_32x16(trow + 16 * h, q);
      }
      // Past the end of the sequence lie the next one's values, or whatever the buffer holds: p is 0 there, but
      // 0 * NaN is not, so those rows of V become zeros
      const int have = t.kv_len - key0;
      bool ok = true;
      if (have < kAttnKeys) {
        const int i = 2 * j + 1, s = i % p.stages;
        ok = warp_wait(full0 + 8 * s, (i / p.stages) & 1, c.status, ATTN_WAIT_KV_TIMEOUT);
        const uint32_t v = ring + s * chunks * kAttnChunkBytes;
        const int vecs = (kAttnKeys - have) * 8;   // 16-byte pieces per chunk
        const int quad = (threadIdx.x >> 5) & 3, first = quad * 32 + (c.tid & 31);
        if (ok)
          for (int ch = 0; ch < chunks; ++ch)
            for (int k = first; k < vecs; k += threads) st_shared_u4(v + ch * kAttnChunkBytes + have * 128 + k * 16, 0, 0, 0, 0);
        fence_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_bar);
      if (!ok) return false;
    }
    m_out = m, l_out = l;
    return true;
  }

  // The slices of a tile become one result (all threads of every CTA of the cluster).
  __device__ __forceinline__ static void join(const Params &p, const TileCtx &c, int split, int slice, int n, int chunks, int rows, int row, bool mine,
                                              bool ok, uint32_t trow, uint32_t area, uint32_t stats_bar, uint32_t join_bar, float m, float l,
                                              uint16_t *out) {
    // every rank's MMAs are done: Q and the ring are free everywhere
    cluster_sync_all();
    if (!mine) return;
    const float mlog = m * p.scale_log2;   // in powers of two
    const uint32_t recv = area + (uint32_t)(split * kAttnRows * 8);
    for (int r = 0; r < split; ++r)
      st_async_f2(peer_smem(area + (uint32_t)(slice * kAttnRows + row) * 8, r), peer_smem(stats_bar, r), mlog, l);
    if (!warp_wait(stats_bar, 0, c.status, ATTN_WAIT_PEERS_TIMEOUT)) ok = false;
    float top = -INFINITY, sum = 0.f;
    for (int r = 0; r < split; ++r) top = fmaxf(top, ld_shared_f2(area + (uint32_t)(r * kAttnRows + row) * 8).x);
    if (top == -INFINITY) top = 0.f;
    for (int r = 0; r < split; ++r) {
      const float2 s = ld_shared_f2(area + (uint32_t)(r * kAttnRows + row) * 8);
      sum += s.y * ex2(s.x - top);
    }
    const float f = l == 0.f ? 0.f : ex2(mlog - top) / sum;
    const int pieces = chunks * 4;   // of 16 columns
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
      const uint32_t dst = peer_smem(slot + (uint32_t)row * 16, ch % split), bar = peer_smem(join_bar, ch % split);
#pragma unroll
      for (int i = 0; i < 4; ++i) st_async_u4(dst + (uint32_t)(i * kAttnRows * 16), bar, r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    }
    if (slice >= pieces) return;   // owns no columns
    if (!warp_wait(join_bar, 0, c.status, ATTN_WAIT_PEERS_TIMEOUT) || !ok || row >= rows) return;
#pragma unroll 1
    for (int ch = slice; ch < pieces; ch += split) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
      for (int r = 0; r < split; ++r) {   // rank order: the sum is deterministic
        const uint32_t src = recv + (uint32_t)((ch / split) * split + r) * (16 * kAttnRows * 4) + (uint32_t)row * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 a = ld_shared_f4(src + (uint32_t)(i * kAttnRows * 16));
          v[4 * i] += a.x, v[4 * i + 1] += a.y, v[4 * i + 2] += a.z, v[4 * i + 3] += a.w;
        }
      }
      store16(out, ch * 16, p.dim, v);
    }
  }
};

}  // namespace bfuse
