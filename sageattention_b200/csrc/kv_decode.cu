// Attention of few query rows per kv head over the 4-bit cache: every key is read once for all of them.
//
//   s_r = scale q_r . k,  p = exp2(s - m),  o_r = sum p v / sum p      over the values that codes and scales stand for
//
// Scores are taken transposed, S^T = K Q^T: the keys are the A operand of mma.sync (m16n8k16, fp16 in, fp32 out), 16 of them per
// instruction, and 8 query rows the B operand; O^T = V^T P^T likewise.  With queries as A 16 rows would be paid for 8.  An E2M1 value times
// its E4M3 scale has 6 significant bits and lies between 2^-10 and 2688, exact in fp16; queries are scaled by a power of two per
// row, so that their 8 bits are exact too (down to 2^-31 of the row's largest).  P is rounded to fp16 once (by 2^-11 at most), with its
// maximum put at 2^6 so that small ones keep their bits down to 2^-20 of it; sums are fp32.
//
// A CTA has four warps; each fetches chunks of 32 keys by cp.async into a ring of its own, so nothing in the loop waits for another warp.
// The four, and then parts of a row that several CTAs have (through a cluster's shared memory, or by a second small kernel, launched as a
// programmatic dependent), are joined by their maxima and sums in a fixed order.
//
// What bounds it: a key costs D 9/8 bytes and, whatever the rows, the instructions that turn its codes into fp16.  32 sequences of 8192 keys, 32
// heads of 8, D=128: 60.8 us, 5.0 TB/s; of 16384 108.8, so that long caches stream at 6.3 (the chip's copy does 6.5) and some 12 us are what
// items cost at their start and end.  Short caches are bound by latency: 1000 keys of one sequence 6.3 us.
#include "kernels.h"
#include "kv_attn.cuh"

namespace sage3 {

namespace {

constexpr int kWarps = 4, kChunk = 32, kStages = 3, kBlock = kWarps * kChunk, kMostParts = 8;

struct Header {                           // at the front of the workspace, for the joining kernel
  int per;                                // units of work per CTA
};

struct Params {
  KvAttnArgs a;
  int group, tiles, page_shift;           // query heads per kv head; tiles of rows of the longest sequence
  int parts, ctas;                        // CTAs of a cluster; of the equal runs
  uint32_t group_inverse;                 // 2^32 / group rounded up: exact for quotients of the few rows there are
  float scale_log2;
  Header* header;
  int* item_start;                        // [B * Hkv, tiles]: number of the item's first unit
  float* o_part;                          // [CTA, 2, rows, DS]
  float2* ml_part;                        // [CTA, 2, rows]: maximum (log2) and sum
  float* lse_add;                         // [B * Hkv, tiles, rows]
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with nothing to add to
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t splat_lo(uint32_t x) { return __byte_perm(x, 0, 0x1010); }
__device__ __forceinline__ uint32_t splat_hi(uint32_t x) { return __byte_perm(x, 0, 0x3232); }
// 128-key blocks of an item (one at least, so that rows without keys are written too) and items per kv head
__device__ __forceinline__ int blocks_of(const KvSeq& s) { return max(1, (s.kv_len + kBlock - 1) / kBlock); }
template <int kRows>
__device__ __forceinline__ int tiles_of(const KvSeq& s, int group) { return (s.q_len * group + kRows - 1) / kRows; }

// shared memory: the rings, and in their place at the end the four warps' results and (clusters) the CTA's own
template <int D, int NB>
struct Smem {
  static constexpr int kRows = 8 * NB, kRing = kWarps * kStages * (kChunk / 16) * 18 * D;
  static constexpr int o = 0, ml = kWarps * kRows * (D + 4) * 4, part = ml + kWarps * kRows * 8, part_ml = part + kRows * D * 4, end = part_ml + kRows * 8;
  static constexpr int bytes = kRing > end ? kRing : end;
};

__device__ __forceinline__ uint32_t of_cta(uint32_t at, int rank) {                     // the same place in the cluster's CTA `rank`
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 ld_cluster(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CTAs per SM that the registers are held to
constexpr int ctas_per_sm(int D, int NB) { return NB == 1 ? 4 : NB == 2 ? 3 : D == 64 && NB == 3 ? 3 : 2; }

// The work: an item is a (sequence, kv head, tile of rows), a unit one of its blocks of 128 keys.  All units, in this order, are dealt out in
// equal runs, so that ragged batches and single long sequences fill the chip alike; a CTA's run may end inside an item and go on to
// others.  Only its first and its last item can be shared with other CTAs: two places for partial results each.
// kCluster, where no item is long beside the others (see plan): a cluster of CTAs has an item, and its parts are joined through their
// shared memory; there is nothing to look up in front and no second kernel.
template <int D, int NB, bool kCluster>   // stored head dim, 8-row blocks
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(D, NB)) kv_decode_kernel(const Params P) {
  using Rec = KvRecord<D>;
  using L = Smem<D, NB>;
  constexpr int kRows = 8 * NB, kRecs = kChunk / 16, kStageBytes = kRecs * Rec::kBytes;
  constexpr int kKS = D / 16;             // k steps of the scores = tiles of 16 channels of the output
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ int scan_s[kWarps], where_s[2];
  __shared__ float add_s[kRows];
  const KvAttnArgs& A = P.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  if (!kCluster) pdl_launch_dependents();

  auto group_of = [&](int row) { return P.group == 1 ? row : (int)__umulhi((uint32_t)row, P.group_inverse); };       // row / group

  // ---- a part of an item: `take` blocks from `block` on (`unit`: the number of its first unit)
  auto item_part = [&](const KvSeq& seq, int b, int h, int tile, int block, int take, int blocks, int unit) {
    const int bh = b * A.Hkv + h;
    const int rows = seq.q_len * P.group, row0 = tile * kRows;
    const int last_row = min(rows, row0 + kRows) - 1;
    const int see_all = seq.seen(A, group_of(row0)), see_any = seq.seen(A, group_of(last_row));   // keys that each row, that any row sees
    const int begin = block * kBlock, end = min(begin + take * kBlock, see_any);
    [[maybe_unused]] const bool whole = take == blocks, head_of_item = block == 0 || kCluster;

    // ---- queries under way: this lane the channels c D/4 ... of row n of each block (used when keys have been asked for: both take as long)
    uint4 q_raw[NB][D / 32];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      const int row = row0 + r * 8 + n, tok = group_of(row), hq = h * P.group + row - tok * P.group;
      const uint4* const src = reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.q + (int64_t)(seq.q0 + tok) * A.q_sn + hq * A.q_sh + c * (D / 4));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        q_raw[r][i] = make_uint4(0, 0, 0, 0);
        if (row < rows && c * (D / 4) + i * 8 < A.D) q_raw[r][i] = __ldg(src + i);
      }
    }

    // ---- keys on their way: chunk number `i` of this warp is keys begin + 32 (kWarps i + warp) ...
    const uint32_t ring = smem_u32(sm) + warp * (kStages * kStageBytes);
    const int chunks = begin < end ? ((end - begin + kChunk - 1) / kChunk - warp + kWarps - 1) / kWarps : 0;
    const int* const table = A.table + b * A.table_stride;
    const int64_t page_bytes = (int64_t)A.Hkv * (A.page_size / 16) * Rec::kBytes;
    const uint8_t* const head = A.data + (int64_t)h * (A.page_size / 16) * Rec::kBytes + lane * 16;
    const bool halves = A.page_size < kChunk;                  // two pages to a chunk
    int ids0 = -1, ids1 = -1;                                  // page ids of 32 chunks, one per lane
    uint32_t absent = 0;                                       // two bits per stage: records whose page there is not
    int in_stage = 0;
    auto fetch = [&](int i) {
      if (i < chunks) {
        const int key = begin + kChunk * (kWarps * i + warp);
        if ((i & 31) == 0) {
          const int mine = key + kBlock * lane;
          ids0 = mine < end ? __ldg(table + (mine >> P.page_shift)) : -1;
          if (halves) ids1 = mine + 16 < end ? __ldg(table + ((mine + 16) >> P.page_shift)) : -1;
        }
        // a record is fetched where its page exists and any of its keys is seen; else it is zeros, and its keys are masked
        const int p0 = __shfl_sync(0xffffffffu, ids0, i & 31);
        const bool ok0 = (uint32_t)p0 < (uint64_t)A.num_pages;
        const uint32_t dst = ring + in_stage * kStageBytes + lane * 16;
        const uint8_t* const r0 = head + (ok0 ? p0 * page_bytes + ((key & (A.page_size - 1)) >> 4) * Rec::kBytes : 0);
        uint32_t none = 0;
        if (!halves && ok0 && key + 16 < end) {
#pragma unroll
          for (int j = 0; j < kStageBytes; j += 512)
            if (j + 512 <= kStageBytes || lane * 16 < kStageBytes - j) cp_async16(dst + j, r0 + j, true);
        } else {
          const int p1 = halves ? __shfl_sync(0xffffffffu, ids1, i & 31) : p0;
          const bool ok1 = (uint32_t)p1 < (uint64_t)A.num_pages && key + 16 < end;
          const uint8_t* const r1 = halves ? head + (ok1 ? p1 * page_bytes : 0) - Rec::kBytes : r0;
#pragma unroll
          for (int j = 0; j < kStageBytes; j += 512)
            if (j + 512 <= kStageBytes || lane * 16 < kStageBytes - j) {
              const bool second = j + lane * 16 >= Rec::kBytes, ok = second ? ok1 : ok0;
              cp_async16(dst + j, ok ? (second ? r1 : r0) + j : head, ok);
            }
          none = (ok0 ? 0u : 1u) | (ok1 ? 0u : 2u);
        }
        absent = (absent & ~(3u << 2 * in_stage)) | none << 2 * in_stage;
        in_stage = in_stage == kStages - 1 ? 0 : in_stage + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i);

    // ---- queries: B fragments
    uint32_t qf[NB][kKS][2];
    float factor[NB][2];                   // of the scores of rows 2 c, 2 c + 1: softmax scale times what undoes the row's power of two
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      uint32_t w[D / 8];
      uint32_t m2 = 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 x = q_raw[r][i];
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        m2 = habsmax2(m2, habsmax2(habsmax2(x.x, x.y), habsmax2(x.z, x.w)));
      }
      m2 = abs2(m2);
      float m = fmaxf(bf16_lo(m2), bf16_hi(m2));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const RowScale scale(m);
      const float up = scale.up, undo = scale.undo;
#pragma unroll
      for (int i = 0; i < kKS; ++i) {
        qf[r][i][0] = pack_f16(bf16_lo(w[2 * i]) * up, bf16_hi(w[2 * i]) * up);
        qf[r][i][1] = pack_f16(bf16_lo(w[2 * i + 1]) * up, bf16_hi(w[2 * i + 1]) * up);
      }
      // (never 0: it multiplies the -inf of masked scores)
      factor[r][0] = fmaxf(__shfl_sync(0xffffffffu, undo, 8 * c) * P.scale_log2, 1.2e-38f);
      factor[r][1] = fmaxf(__shfl_sync(0xffffffffu, undo, 8 * c + 4) * P.scale_log2, 1.2e-38f);
      if (A.lse != nullptr && head_of_item && warp == 0) {     // scores of the keys with their offset: scale q . offset more
        float s = 0.f;
        if (A.k_offset != nullptr) {
          const __nv_bfloat16* const off = (const __nv_bfloat16*)A.k_offset + (int64_t)h * A.D + c * (D / 4);
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
            if (c * (D / 4) + i * 8 < A.D) {
              const uint4 x = __ldg(reinterpret_cast<const uint4*>(off) + i);
              const uint32_t o[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) s = fmaf(bf16_lo(w[4 * i + j]), bf16_lo(o[j]), fmaf(bf16_hi(w[4 * i + j]), bf16_hi(o[j]), s));
            }
          s += __shfl_xor_sync(0xffffffffu, s, 1);
          s += __shfl_xor_sync(0xffffffffu, s, 2);
        }
        if (c == 0) add_s[r * 8 + n] = s * A.sm_scale;
      }
    }
    int limit[NB][2];                      // keys that rows 2 c, 2 c + 1 see
#pragma unroll
    for (int r = 0; r < NB; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = row0 + r * 8 + 2 * c + j;
        limit[r][j] = row < rows ? seq.seen(A, group_of(row)) : 0;
      }

    float o[kKS][NB][4];
    float2 m_row[NB], l_row[NB];           // of rows 2 c, 2 c + 1: what stands for the maximum, and this lane's part of the sum
#pragma unroll
    for (int r = 0; r < NB; ++r) {
#pragma unroll
      for (int i = 0; i < kKS; ++i) o[i][r][0] = o[i][r][1] = o[i][r][2] = o[i][r][3] = 0.f;
      m_row[r] = make_float2(kLowest, kLowest);
      l_row[r] = make_float2(0.f, 0.f);
    }

    int stage = 0;
#pragma unroll 1
    for (int i = 0; i < chunks; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();                        // every lane's part of chunk i is here, and chunk i - 1 has been read by all
      const uint32_t gone = absent >> 2 * stage & 3u;
      fetch(i + kStages - 1);
      const uint32_t st = ring + stage * kStageBytes;
      stage = stage == kStages - 1 ? 0 : stage + 1;
      const int key0 = begin + kChunk * (kWarps * i + warp);

      float s[kRecs][NB][4];
#pragma unroll
      for (int g = 0; g < kRecs; ++g) {
        const uint32_t rec = st + g * Rec::kBytes;
        uint32_t ka[D / 32], kb[D / 32], sa[2], sb[2];          // codes and scales of tokens n, n + 8
        if constexpr (D == 128) {
          const uint4 x = lds128(rec + lane * 16), y = lds128(rec + 512 + lane * 16);
          ka[0] = x.x; ka[1] = x.y; ka[2] = x.z; ka[3] = x.w;
          kb[0] = y.x; kb[1] = y.y; kb[2] = y.z; kb[3] = y.w;
          const uint32_t sc = lds32(rec + Rec::kKeyScales + lane * 4);
          const uint32_t f0 = e4m3x2_to_f16(sc), f1 = e4m3x2_to_f16(sc >> 16);
          sa[0] = splat_lo(f0); sa[1] = splat_hi(f0); sb[0] = splat_lo(f1); sb[1] = splat_hi(f1);
        } else {
          const uint2 x = lds64(rec + lane * 8), y = lds64(rec + 256 + lane * 8);
          ka[0] = x.x; ka[1] = x.y; kb[0] = y.x; kb[1] = y.y;
          const uint32_t f = e4m3x2_to_f16(lds16(rec + Rec::kKeyScales + lane * 2));
          sa[0] = sa[1] = splat_lo(f); sb[0] = sb[1] = splat_hi(f);
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t x[4], y[4];
          e2m1x8_to_f16(ka[w], x);
          e2m1x8_to_f16(kb[w], y);
          const int blk = D == 128 ? w / 2 : 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) { x[j] = hmul2(x[j], sa[blk]); y[j] = hmul2(y[j], sb[blk]); }
#pragma unroll
          for (int r = 0; r < NB; ++r) {
            if (w == 0) mma_f16_first(s[g][r], x[0], y[0], x[1], y[1], qf[r][0][0], qf[r][0][1]);
            else mma_f16(s[g][r], x[0], y[0], x[1], y[1], qf[r][2 * w][0], qf[r][2 * w][1]);
            mma_f16(s[g][r], x[2], y[2], x[3], y[3], qf[r][2 * w + 1][0], qf[r][2 * w + 1][1]);
          }
        }
      }

      uint32_t vsc[kRecs];                 // E4M3 of block n (n / 2) and tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
      for (int g = 0; g < kRecs; ++g)
        vsc[g] = lds32(st + g * Rec::kBytes + Rec::kValueScales + (D == 128 ? lane * 4 : (lane >> 3) * 16 + c * 4));

      if (key0 + kChunk > see_all || gone != 0) {
#pragma unroll
        for (int g = 0; g < kRecs; ++g) {
          // Values that no row sees add nothing, whatever lies there.  A NaN scale among the values (E4M3 has no other such code)
          // must not reach rows that do not see its key, so it goes by way of the scores of those that do.
          uint32_t nan_keys[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (key0 + g * 16 + 2 * c + (j & 1) + (j >> 1) * 8 >= see_any || (gone >> g & 1)) vsc[g] &= ~(0xffu << (8 * j));
            const bool bad = (vsc[g] >> (8 * j) & 0x7fu) == 0x7fu;
            nan_keys[j] = __ballot_sync(0xffffffffu, bad) & (0x11111111u << (n >> 1));
            if (bad) vsc[g] &= ~(0xffu << (8 * j));
          }
#pragma unroll
          for (int r = 0; r < NB; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if ((n & 1 ? nan_keys[(j & 2) + 1] : nan_keys[j & 2]) != 0) s[g][r][j] = NAN;
              if (key0 + g * 16 + n + (j >> 1) * 8 >= limit[r][j & 1] || (gone >> g & 1)) s[g][r][j] = -INFINITY;
            }
        }
      }

      // ---- P.  exp2's arguments against the maximum as it stands; where one is too large for fp16, the maxima are brought up to
      // date first (hardly ever after the first chunks, so that no lane asks another in the others)
      uint32_t p[kRecs][NB][2];
#pragma unroll
      for (int r = 0; r < NB; ++r) {
        const float2 f = make_float2(factor[r][0], factor[r][1]);
        float2 e[kRecs][2];
        float top = kLowest;
        auto arguments = [&]() {
          const float2 base = make_float2(kTop - m_row[r].x, kTop - m_row[r].y);
#pragma unroll
          for (int g = 0; g < kRecs; ++g)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              e[g][j] = ffma2(make_float2(s[g][r][2 * j], s[g][r][2 * j + 1]), f, base);
              top = fmaxf(top, fmaxf(e[g][j].x, e[g][j].y));
            }
        };
        arguments();
        if (__any_sync(0xffffffffu, top > kTop + kSlack)) {
          float2 m = m_row[r];
#pragma unroll
          for (int g = 0; g < kRecs; ++g) {
            m.x = fmaxf(m.x, fmaxf(s[g][r][0], s[g][r][2]) * f.x);
            m.y = fmaxf(m.y, fmaxf(s[g][r][1], s[g][r][3]) * f.y);
          }
#pragma unroll
          for (int d = 4; d < 32; d *= 2) {
            m.x = fmaxf(m.x, __shfl_xor_sync(0xffffffffu, m.x, d));
            m.y = fmaxf(m.y, __shfl_xor_sync(0xffffffffu, m.y, d));
          }
          const float2 corr = make_float2(ex2_approx(m_row[r].x - m.x), ex2_approx(m_row[r].y - m.y));
          m_row[r] = m;
          l_row[r].x *= corr.x; l_row[r].y *= corr.y;
#pragma unroll
          for (int k = 0; k < kKS; ++k) {
            o[k][r][0] *= corr.x; o[k][r][1] *= corr.y; o[k][r][2] *= corr.x; o[k][r][3] *= corr.y;
          }
          arguments();
        }
#pragma unroll
        for (int g = 0; g < kRecs; ++g)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = make_float2(ex2_approx(e[g][j].x), ex2_approx(e[g][j].y));
            l_row[r] = fadd2(l_row[r], x);
            p[g][r][j] = transpose8x8(pack_f16(x.x, x.y));
          }
      }

      // ---- O^T += V^T P^T: the codes of two tokens of a channel go to one byte, whose conversion then gives the fragment's pair
#pragma unroll
      for (int g = 0; g < kRecs; ++g) {
        const uint32_t rec = st + g * Rec::kBytes + Rec::kValues;
        const uint32_t sv[2] = {e4m3x2_to_f16(vsc[g]), e4m3x2_to_f16(vsc[g] >> 16)};
        uint32_t v0[2][D / 64], v1[2][D / 64];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          if constexpr (D == 128) {
            const uint4 x = lds128(rec + hh * 512 + lane * 16);
            v0[hh][0] = x.x; v0[hh][1] = x.y; v1[hh][0] = x.z; v1[hh][1] = x.w;
          } else {
            const uint2 x = lds64(rec + hh * 256 + lane * 8);
            v0[hh][0] = x.x; v1[hh][0] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 64; ++w) {
          uint32_t even[2][4], odd[2][4];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const uint32_t x = v0[hh][w], y = v1[hh][w];
            e2m1x8_to_f16((x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u), even[hh]);
            e2m1x8_to_f16(((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u), odd[hh]);
#pragma unroll
            for (int j = 0; j < 4; ++j) { even[hh][j] = hmul2(even[hh][j], sv[hh]); odd[hh][j] = hmul2(odd[hh][j], sv[hh]); }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < NB; ++r) mma_f16(o[4 * w + j][r], even[0][j], odd[0][j], even[1][j], odd[1][j], p[g][r][0], p[g][r][1]);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    if (!kCluster && head_of_item && threadIdx.x == 0) P.item_start[(int64_t)bh * P.tiles + tile] = unit;

    // ---- join the four warps
    __syncthreads();
    float* const o_s = reinterpret_cast<float*>(sm + L::o);               // [warp][row][D + 4]
    float2* const ml_s = reinterpret_cast<float2*>(sm + L::ml);
#pragma unroll
    for (int r = 0; r < NB; ++r) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = j == 0 ? l_row[r].x : l_row[r].y;
#pragma unroll
        for (int d = 4; d < 32; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
        const int row = r * 8 + 2 * c + j;
        float* const dst = o_s + (warp * kRows + row) * (D + 4) + n * (D / 8);
#pragma unroll
        for (int k = 0; k < kKS; k += 2)
          *reinterpret_cast<float4*>(dst + 2 * k) = make_float4(o[k][r][j], o[k][r][2 + j], o[k + 1][r][j], o[k + 1][r][2 + j]);
        if (n == 0) ml_s[warp * kRows + row] = make_float2(j == 0 ? m_row[r].x : m_row[r].y, l);
      }
    }
    __syncthreads();
    constexpr int kPer = D / 32;                                          // channels of a row per lane; a warp has every fourth row
#pragma unroll 1
    for (int row = warp; row < kRows && row0 + row < rows; row += kWarps) {
      float m = kLowest, l = 0.f, wgt[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml_s[w * kRows + row].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 x = ml_s[w * kRows + row];
        wgt[w] = ex2_approx(x.x - m);
        l += wgt[w] * x.y;
      }
      float acc[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
#pragma unroll
        for (int k = 0; k < kPer; k += 2) {
          const float2 x = *reinterpret_cast<const float2*>(o_s + (w * kRows + row) * (D + 4) + lane * kPer + k);
          acc[k] = fmaf(wgt[w], x.x, acc[k]); acc[k + 1] = fmaf(wgt[w], x.y, acc[k + 1]);
        }
      if constexpr (kCluster) {
#pragma unroll
        for (int k = 0; k < kPer; k += 2) reinterpret_cast<float2*>(sm + L::part)[(row * D + lane * kPer + k) / 2] = make_float2(acc[k], acc[k + 1]);
        if (lane == 0) reinterpret_cast<float2*>(sm + L::part_ml)[row] = make_float2(m, l);
      } else {
        const int tok = group_of(row0 + row), hq = h * P.group + row0 + row - tok * P.group;
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.0f / l;
          __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh + lane * kPer;
          if (lane * kPer < A.D)
#pragma unroll
            for (int k = 0; k < kPer; k += 2) *reinterpret_cast<uint32_t*>(out + k) = pack_bf16(acc[k] * inv, acc[k + 1] * inv);
          if (lane == 0 && A.lse != nullptr) A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = lse_of(m, l, add_s[row]);
        } else {
          const int64_t at = ((int64_t)blockIdx.x * 2 + (head_of_item ? 1 : 0)) * kRows + row;
#pragma unroll
          for (int k = 0; k < kPer; k += 2) *reinterpret_cast<float2*>(P.o_part + at * D + lane * kPer + k) = make_float2(acc[k], acc[k + 1]);
          if (lane == 0) P.ml_part[at] = make_float2(m, l);
          if (lane == 0 && head_of_item && A.lse != nullptr) P.lse_add[((int64_t)bh * P.tiles + tile) * kRows + row] = add_s[row];
        }
      }
    }
  };

  if constexpr (kCluster) {
    const int item = blockIdx.x / P.parts, part = blockIdx.x - item * P.parts, bh = item / P.tiles, tile = item - bh * P.tiles;
    const int b = bh / A.Hkv, h = bh - b * A.Hkv;
    const KvSeq seq(A, b);
    const int rows = seq.q_len * P.group, row0 = tile * kRows;
    // Nobody leaves before the last barrier, and barriers do not hang on what a warp has read: lengths that another stream writes meanwhile may
    // differ from CTA to CTA, and a CTA that has gone must not be read from.
    const bool live = __syncthreads_and(row0 < rows);
    if (live) {
      const int blocks = blocks_of(seq), per = (blocks + P.parts - 1) / P.parts, block = min(part * per, blocks);
      item_part(seq, b, h, tile, block, min(per, blocks - block), blocks, 0);
    }
    __syncwarp();
    cluster_sync();
    // rows dealt out to the CTAs' warps, parts in the order of the keys
    constexpr int kPer = D / 32;
    const uint32_t at_o = smem_u32(sm + L::part), at_ml = smem_u32(sm + L::part_ml);
    const bool have = lane * kPer < A.D;
#pragma unroll 1
    for (int row = part + P.parts * warp; live && row < kRows && row0 + row < rows; row += P.parts * kWarps) {
      float2 ml = make_float2(kLowest, 0.f);
      if (lane < P.parts) ml = ld_cluster(of_cta(at_ml + row * 8, lane));
      float m = ml.x;
#pragma unroll
      for (int d = 4; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      m = __shfl_sync(0xffffffffu, m, 0);
      const float mine = ex2_approx(ml.x - m);
      float acc[kPer], l = 0.f;
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
#pragma unroll
      for (int x = 0; x < kMostParts; ++x) {
        const float w = __shfl_sync(0xffffffffu, mine, x), lx = __shfl_sync(0xffffffffu, ml.y, x);
        if (x < P.parts) {
          l = fmaf(w, lx, l);
#pragma unroll
          for (int k = 0; k < kPer; k += 2) {
            if (!have) continue;           // (a load that nothing waits for could be under way when its target goes)
            const float2 v = ld_cluster(of_cta(at_o + (row * D + lane * kPer + k) * 4, x));
            acc[k] = fmaf(w, v.x, acc[k]); acc[k + 1] = fmaf(w, v.y, acc[k + 1]);
          }
        }
      }
      const int tok = group_of(row0 + row), hq = h * P.group + row0 + row - tok * P.group;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh + lane * kPer;
      if (have)
#pragma unroll
        for (int k = 0; k < kPer; k += 2) *reinterpret_cast<uint32_t*>(out + k) = pack_bf16(acc[k] * inv, acc[k + 1] * inv);
      if (lane == 0 && A.lse != nullptr) A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = lse_of(m, l, add_s[row]);
    }
    __syncwarp();
    cluster_sync();                        // nobody's shared memory goes while another reads it
  } else {
    // ---- this CTA's units
    auto units = [&](int b) {
      const KvSeq s(A, b);
      return A.Hkv * tiles_of<kRows>(s, P.group) * blocks_of(s);
    };
    // a thread has some sequences next to one another; one scan gives it the units in front of them, and their total
    const int each = (A.B + kWarps * 32 - 1) / (kWarps * 32), b_first = min((int)threadIdx.x * each, A.B), b_last = min(b_first + each, A.B);
    int mine = 0;
    for (int b = b_first; b < b_last; ++b) mine += units(b);
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += x;
    }
    if (lane == 31) scan_s[warp] = incl;
    __syncthreads();
    int total = 0, before = incl - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan_s[w];
      total += scan_s[w];
    }
    const int per = (int)(((uint32_t)total + gridDim.x - 1) / gridDim.x);
    int unit = blockIdx.x * per;
    const int unit_end = min(unit + per, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) P.header->per = per;
    if (unit >= unit_end) return;
    if (unit >= before && unit < before + mine) {                // one of this thread's is the first
      int b = b_first, x = before;
      for (int n_b; b + 1 < b_last && unit >= x + (n_b = units(b)); ++b) x += n_b;
      where_s[0] = b; where_s[1] = x;
    }
    __syncthreads();
    int b = where_s[0];
    int rest = unit - where_s[1];            // units of sequence b before this one

    // Each round has the same barriers for all warps and ends by a vote, so that all take as many, whatever each has read of lengths that another
    // stream writes meanwhile.
#pragma unroll 1
    do {
      for (;;) {
        const KvSeq seq(A, b);
        const int blocks = blocks_of(seq), tiles = tiles_of<kRows>(seq, P.group);
        if (rest >= A.Hkv * tiles * blocks) {           // on to the next sequence
          rest -= A.Hkv * tiles * blocks;
          if (++b < A.B) continue;
          unit = unit_end;                               // (there is none: lengths have changed)
          __syncthreads();                               // as in an item
          __syncthreads();
          break;
        }
        const int item = rest / blocks, block = rest - item * blocks, take = min(blocks - block, unit_end - unit), h = item / tiles, tile = item - h * tiles;
        item_part(seq, b, h, tile, block, take, blocks, unit);
        unit += take;
        rest += take;
        break;
      }
    } while (__syncthreads_and(unit < unit_end));        // (and the ring is the next item's)
  }
}

// Items that more than one CTA had, in the order of the keys: a warp per row, a lane D / 32 channels.  kWide, where few items have many parts
// each: four warps per row, which take four parts each in turn (B2 131072 keys, 37 parts each: 66.7 -> 61.4 us; B1 8192 keys 16.3 -> 10.8).
template <int D, int NB, bool kWide>
__global__ void __launch_bounds__(128) kv_join_kernel(const Params P) {
  constexpr int kRows = 8 * NB, V = D / 32;
  const KvAttnArgs& A = P.a;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const uint32_t id = kWide ? blockIdx.x : blockIdx.x * 4 + warp, item = id / kRows;
  const int row_id = id % kRows, bh = item / P.tiles, tile = item - bh * P.tiles;
  if (bh >= A.B * A.Hkv) return;                                // (a whole warp; others of the CTA wait below)
  const int b = bh / A.Hkv, h = bh - b * A.Hkv;
  const KvSeq seq(A, b);
  const int row = tile * kRows + row_id;
  pdl_wait();                              // also where there is no row: what follows on the stream may write the first kernel's inputs
  if (row >= seq.q_len * P.group) return;
  // (held to the parts that there are, should lengths have changed since the first kernel read them)
  const uint32_t start = P.item_start[item], per = max(P.header->per, 1), most = P.ctas - 1;
  const int first = min(start / per, most), last = min((start + blocks_of(seq) - 1) / per, most);
  if (first == last) return;
  // the first CTA had the item last, the others had it first
  auto place = [&](int cta) { return ((int64_t)cta * 2 + (cta == first ? 1 : 0)) * kRows + row_id; };
  // four parts at a time, all of them loaded before the first is used
  constexpr int kAtOnce = 4;
  float acc[V], l = 0.f, m = kLowest;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 1
  for (int x = first + (kWide ? warp * kAtOnce : 0); x <= last; x += kAtOnce * (kWide ? 4 : 1)) {
    float2 ml[kAtOnce];
    float v[kAtOnce][V];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      ml[y] = make_float2(kLowest, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) v[y][i] = 0.f;
      if (x + y <= last) {
        const int64_t at = place(x + y);
        ml[y] = P.ml_part[at];
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float2 u = *reinterpret_cast<const float2*>(P.o_part + at * D + lane * V + i);
          v[y][i] = u.x; v[y][i + 1] = u.y;
        }
      }
    }
    float top = m;
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) top = fmaxf(top, ml[y].x);
    const float old = ex2_approx(m - top);
    m = top;
    l *= old;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] *= old;
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const float w = ex2_approx(ml[y].x - m);
      l = fmaf(w, ml[y].y, l);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(w, v[y][i], acc[i]);
    }
  }
  if (kWide) {
    __shared__ float part_s[4][D + 2];
#pragma unroll
    for (int i = 0; i < V; ++i) part_s[warp][lane * V + i] = acc[i];
    if (lane == 0) { part_s[warp][D] = m; part_s[warp][D + 1] = l; }
    __syncthreads();
    if (warp != 0) return;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, part_s[w][D]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float wgt = ex2_approx(part_s[w][D] - m);
      l = fmaf(wgt, part_s[w][D + 1], l);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(wgt, part_s[w][lane * V + i], acc[i]);
    }
  }
  const int tok = row / P.group, hq = h * P.group + row - tok * P.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh + lane * V;
  if (lane * V < A.D) {
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16(acc[i] * inv, acc[i + 1] * inv);
  }
  if (lane == 0 && A.lse != nullptr)
    A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = lse_of(m, l, P.lse_add[(int64_t)item * kRows + row_id]);
}

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

struct Plan {
  int nb, tiles;
  int parts;                              // CTAs of a cluster; 0: equal runs
  int64_t ctas, units, rows;              // units and rows (padded to tiles), counted in 32 bits by the kernels
  size_t starts, adds, ml, o;             // offsets in the workspace
  size_t bytes;
};

// Up to 24 (D=64: 32) rows at a time, in tiles as equal as can be; as many CTAs as fit on the chip at once, or as there are units.
Plan plan(int B, int Hq, int Hkv, int DS, int max_q, int max_k, int sms) {
  Plan p{};
  const int64_t rows = (int64_t)max_q * (Hq / Hkv), most = DS == 64 ? 32 : 24;
  p.tiles = (int)((rows + most - 1) / most);
  p.nb = (int)((rows + 8 * p.tiles - 1) / (8 * p.tiles));
  const int64_t items = (int64_t)B * Hkv * p.tiles, blocks = ((int64_t)max_k + kBlock - 1) / kBlock;
  const int64_t fit = (int64_t)sms * ctas_per_sm(DS, p.nb);
  p.units = items * blocks;
  p.rows = items * 8 * p.nb;
  p.ctas = p.units < fit ? p.units : fit;
  // A cluster (or a CTA) per item or equal runs?  Clusters are as large as all of them fit at once; a CTA's way through the keys must not be
  // long beside an equal share of all of them, nor the last round of CTAs nearly empty.  us, equal runs -> clusters, lengths up to what is said, one
  // token unless it says more.  32 heads of 8, D=128: B1 1000 keys 6.6 -> 6.7, B4 8192 15.1 -> 13.9, B12 4096 16.6 -> 14.1, B32 2048 17.6 -> 16.0,
  // B64 1000 20.4 -> 15.9, B256 1000 57.8 -> 49.4, B128 1000 of 4 tokens 52.4 -> 48.6; D=64: B12 4096 12.8 -> 10.5, B64 1000 15.8 -> 11.5, B256 1000
  // 40.6 -> 35.2; 16 heads of 16: B64 1000 D=128 31.1 -> 27.0, D=64 22.5 -> 19.5; 8 heads of 1, D=128: B256 1000 16.6 -> 12.3.
  // What the rule leaves to equal runs: 32 heads of 8, B1 16384 12.5 -> 18.1, B40 8192 48.5 -> 68.2, D=64 32.9 -> 47.2; 16 heads of 16, B1 16384 15.0 ->
  // 21.6; 8 heads of 1, B4 8192 9.2 -> 12.3.  Of 46 such shapes it takes the slower one by 8 % at most (8 heads of 1, B12 4096: 9.1 in place of 8.4).
  // One block needs no joining (4.1 -> 4.6).
  p.parts = kMostParts;
  while (p.parts > 1 && (items * p.parts > fit || p.parts >= 2 * blocks)) p.parts /= 2;
  const int64_t longest = (blocks + p.parts - 1) / p.parts;
  const bool clusters = items <= fit ? longest <= 16 && (longest - 7) * fit <= p.units : longest <= 32 && 10 * items >= 13 * fit;
  if (blocks < 2 || !clusters) p.parts = 0;
  p.starts = 256;
  p.adds = p.starts + align256(items * 4);
  p.ml = p.adds + align256(items * 8 * p.nb * 4);
  p.o = p.ml + align256(p.ctas * 2 * 8 * p.nb * 8);
  p.bytes = p.parts != 0 ? 0 : p.o + align256(p.ctas * 2 * 8 * p.nb * DS * 4);
  return p;
}

template <int D, int NB>
cudaError_t launch(const Params& P, const Plan& p, bool split, cudaStream_t stream) {
  constexpr int smem = Smem<D, NB>::bytes;
  if (p.parts != 0) {
    static std::atomic<uint64_t> allowed;
    if (cudaError_t e = allow_smem(kv_decode_kernel<D, NB, true>, smem, allowed); e != cudaSuccess) return e;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(P.a.B * P.a.Hkv * P.tiles * p.parts)); c.blockDim = dim3(kWarps * 32); c.dynamicSmemBytes = smem; c.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = p.parts; at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at; c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kv_decode_kernel<D, NB, true>, P);
  }
  static std::atomic<uint64_t> allowed;
  if (cudaError_t e = allow_smem(kv_decode_kernel<D, NB, false>, smem, allowed); e != cudaSuccess) return e;
  if (cudaError_t e = launch_pdl(kv_decode_kernel<D, NB, false>, dim3((unsigned)p.ctas), kWarps * 32, smem, stream, false, P); e != cudaSuccess) return e;
  if (!split) return cudaGetLastError();
  const int64_t items = (int64_t)P.a.B * P.a.Hkv * P.tiles, rows = items * 8 * NB;
  if (items * 8 <= p.ctas) return launch_pdl(kv_join_kernel<D, NB, true>, dim3((unsigned)rows), 128, 0, stream, true, P);
  return launch_pdl(kv_join_kernel<D, NB, false>, dim3((unsigned)((rows + 3) / 4)), 128, 0, stream, true, P);
}

}  // namespace

size_t kv_decode_workspace(int B, int Hq, int Hkv, int DS, int max_q, int max_k, int sms) { return plan(B, Hq, Hkv, DS, max_q, max_k, sms).bytes; }

bool kv_decode_fits(int B, int Hq, int Hkv, int max_q, int max_k) {
  const Plan p = plan(B, Hq, Hkv, 128, max_q, max_k, 1);
  return p.units < (1ll << 30) && p.rows < (1ll << 30);
}

cudaError_t launch_kv_decode(const KvAttnArgs& a, cudaStream_t stream) {
  int sms;
  if (cudaError_t e = sm_count(&sms); e != cudaSuccess) return e;
  const Plan p = plan(a.B, a.Hq, a.Hkv, a.DS, a.max_q, a.max_k, sms);
  if (p.units >= (1ll << 30) || p.rows >= (1ll << 30)) return cudaErrorInvalidValue;      // (kv_decode_fits has said so)
  Params P;
  P.a = a;
  P.group = a.Hq / a.Hkv; P.tiles = p.tiles;
  P.group_inverse = (uint32_t)(0xffffffffu / (uint32_t)P.group) + 1;
  P.scale_log2 = a.sm_scale * kLog2e;
  P.parts = p.parts; P.ctas = (int)p.ctas;
  P.page_shift = 0;
  while ((1 << P.page_shift) < a.page_size) ++P.page_shift;
  P.header = nullptr; P.item_start = nullptr; P.lse_add = nullptr; P.ml_part = nullptr; P.o_part = nullptr;
  if (p.bytes != 0) {
    char* const w = (char*)a.workspace;
    P.header = (Header*)w;
    P.item_start = (int*)(w + p.starts); P.lse_add = (float*)(w + p.adds);
    P.ml_part = (float2*)(w + p.ml); P.o_part = (float*)(w + p.o);
  }
  const bool split = a.max_k > kBlock;     // else an item is one unit
  if (a.DS == 128) return p.nb == 1 ? launch<128, 1>(P, p, split, stream) : p.nb == 2 ? launch<128, 2>(P, p, split, stream) : launch<128, 3>(P, p, split, stream);
  return p.nb == 1   ? launch<64, 1>(P, p, split, stream)
         : p.nb == 2 ? launch<64, 2>(P, p, split, stream)
         : p.nb == 3 ? launch<64, 3>(P, p, split, stream)
                     : launch<64, 4>(P, p, split, stream);
}

}  // namespace sage3
