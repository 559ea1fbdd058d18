// Attention of few query rows per kv head over the 4-bit cache: every key is read once for all of them.
//
//   s_r = scale q_r . k,  p = exp2(s - m),  o_r = sum p v / sum p      over the values that codes and scales stand for
//
// Scores are taken transposed, S^T = K Q^T: the keys are the A operand of mma.sync (m16n8k16, fp16 in, fp32 out), 16 of them per
// instruction, and 8 query rows the B operand; O^T = V^T P^T likewise.  With queries as A 16 rows would be paid for 8.  An E2M1 value times
// its E4M3 scale has 6 significant bits and lies between 2^-10 and 2688, exact in fp16; queries are scaled by a power of two per
// row, so that their 8 bits are exact too (down to 2^-31 of the row's largest).  P is rounded to fp16 once (2^-12 relative), with its
// maximum put at 2^8 so that small ones keep their bits down to 2^-22 of it; sums are fp32.
//
// A CTA of four warps takes a (sequence, kv head, 8 or 16 rows, range of keys); each warp fetches chunks of 32 keys by cp.async into a
// ring of its own, so nothing in the loop waits for another warp.  The four and then the ranges (a second small kernel, launched
// as a programmatic dependent) are joined by their maxima and sums in a fixed order.
#include "kernels.h"
#include "kv_cache.cuh"

namespace sage3 {

namespace {

constexpr int kWarps = 4, kChunk = 32, kStages = 3;
constexpr float kTop = 8.f;               // log2 of the largest P

struct Params {
  KvAttnArgs a;
  int group, rows_per_tile, tiles, splits, split_keys, page_shift;
  float scale_log2;
  float* o_part;                          // [B * Hkv, tiles, splits, rows, DS]
  float2* ml_part;                        // [B * Hkv, tiles, splits, rows]: maximum (log2) and sum
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t splat_lo(uint32_t x) { return __byte_perm(x, 0, 0x1010); }
__device__ __forceinline__ uint32_t splat_hi(uint32_t x) { return __byte_perm(x, 0, 0x3232); }
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}

// Where a sequence's rows and keys lie; every bound that memory accesses rely on is taken here.
struct Seq {
  int q0, q_len, kv_len;
  __device__ __forceinline__ Seq(const KvAttnArgs& A, int b) {
    q0 = b; q_len = 1;
    if (A.cu_q != nullptr) { q0 = __ldg(A.cu_q + b); q_len = __ldg(A.cu_q + b + 1) - q0; }
    if (q0 < 0 || q_len < 0 || q0 > A.tokens) { q0 = 0; q_len = 0; }
    q_len = min(min(q_len, A.max_q), A.tokens - q0);
    kv_len = (int)min((int64_t)max(__ldg(A.kv_lens + b), 0), (int64_t)A.cols * A.page_size);
    kv_len = min(kv_len, A.max_k);
  }
  // keys that token t of the sequence sees
  __device__ __forceinline__ int seen(const KvAttnArgs& A, int t) const { return A.causal ? max(0, min(kv_len, kv_len - q_len + t + 1)) : kv_len; }
};

template <int D, int NB>
constexpr int smem_bytes() {
  return kWarps * kStages * (kChunk / 16) * 18 * D > kWarps * 8 * NB * ((D + 4) * 4 + 8) ? kWarps * kStages * (kChunk / 16) * 18 * D
                                                                                        : kWarps * 8 * NB * ((D + 4) * 4 + 8);
}

template <int D, int NB>                  // stored head dim, 8-row blocks
__global__ void __launch_bounds__(kWarps * 32, NB == 1 ? 4 : 3) kv_decode_kernel(const Params P) {
  using Rec = KvRecord<D>;
  constexpr int kRows = 8 * NB, kRecs = kChunk / 16, kStageBytes = kRecs * Rec::kBytes;
  constexpr int kKS = D / 16;             // k steps of the scores = tiles of 16 channels of the output
  extern __shared__ __align__(16) uint8_t sm[];
  const KvAttnArgs& A = P.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
  const int bh = blockIdx.x, b = bh / A.Hkv, h = bh - b * A.Hkv, tile = blockIdx.y, split = blockIdx.z;
  pdl_launch_dependents();
  const Seq seq(A, b);
  const int rows = seq.q_len * P.group, row0 = tile * kRows;
  if (row0 >= rows) return;
  const int last_row = min(rows, row0 + kRows) - 1;
  const int see_all = seq.seen(A, row0 / P.group), see_any = seq.seen(A, last_row / P.group);   // keys that each row, that any row sees
  const int begin = split * P.split_keys, end = min(begin + P.split_keys, see_any);
  if (begin >= end && (split > 0 || P.splits > 1)) return;

  // ---- keys on their way: chunk number `i` of this warp is keys begin + 32 (kWarps i + warp) ...
  const uint32_t ring = smem_u32(sm) + warp * (kStages * kStageBytes);
  const int chunks = begin < end ? ((end - begin + kChunk - 1) / kChunk - warp + kWarps - 1) / kWarps : 0;
  const int* const table = A.table + b * A.table_stride;
  const int64_t page_bytes = (int64_t)A.Hkv * (A.page_size / 16) * Rec::kBytes;
  const uint8_t* const head = A.data + (int64_t)h * (A.page_size / 16) * Rec::kBytes;
  const bool halves = A.page_size < kChunk;                    // two pages to a chunk
  int ids0 = -1, ids1 = -1;                                    // page ids of 32 chunks, one per lane
  uint32_t absent = 0;                                         // two bits per stage: records whose page there is not
  auto fetch = [&](int i) {
    if (i < chunks) {
      if ((i & 31) == 0) {
        const int key = begin + kChunk * (kWarps * (i + lane) + warp);
        ids0 = key < end ? __ldg(table + (key >> P.page_shift)) : -1;
        if (halves) ids1 = key + 16 < end ? __ldg(table + ((key + 16) >> P.page_shift)) : -1;
      }
      const int key = begin + kChunk * (kWarps * i + warp);
      const int p0 = __shfl_sync(0xffffffffu, ids0, i & 31), p1 = halves ? __shfl_sync(0xffffffffu, ids1, i & 31) : p0;
      // a record is fetched where its page exists and any of its keys is seen; else it is zeros, and its keys are masked
      const bool ok0 = p0 >= 0 && p0 < A.num_pages, ok1 = p1 >= 0 && p1 < A.num_pages && key + 16 < end;
      const int in0 = (key & (A.page_size - 1)) >> 4;
      const uint8_t* const r0 = head + (ok0 ? p0 * page_bytes + in0 * Rec::kBytes : 0);
      const uint8_t* const r1 = head + (ok1 ? p1 * page_bytes + (halves ? 0 : in0 + 1) * Rec::kBytes : 0) - Rec::kBytes;
      const uint32_t dst = ring + (i % kStages) * kStageBytes;
      absent = (absent & ~(3u << 2 * (i % kStages))) | ((ok0 ? 0u : 1u) | (ok1 ? 0u : 2u)) << 2 * (i % kStages);
#pragma unroll
      for (int j = 0; j < kStageBytes; j += 512) {
        const int at = j + lane * 16;
        const bool second = at >= Rec::kBytes;
        if (kStageBytes % 512 == 0 || at < kStageBytes)
          cp_async16(dst + at, (second ? (ok1 ? r1 + at : head) : (ok0 ? r0 + at : head)), second ? ok1 : ok0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  // ---- queries: B fragments, this lane the channels c D/4 ... of row n of each block
  uint32_t qf[NB][kKS][2];
  float factor[NB][2];                     // of the scores of rows 2 c, 2 c + 1: softmax scale times what undoes the row's power of two
  float lse_add[NB];                       // row n
#pragma unroll
  for (int r = 0; r < NB; ++r) {
    const int row = row0 + r * 8 + n, tok = row / P.group, hq = h * P.group + row - tok * P.group;
    const __nv_bfloat16* const src = (const __nv_bfloat16*)A.q + (int64_t)(seq.q0 + tok) * A.q_sn + hq * A.q_sh + c * (D / 4);
    uint32_t w[D / 8];
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row < rows && c * (D / 4) + i * 8 < A.D) x = __ldg(reinterpret_cast<const uint4*>(src) + i);
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      m2 = habsmax2(m2, habsmax2(habsmax2(x.x, x.y), habsmax2(x.z, x.w)));
    }
    m2 = abs2(m2);
    float m = fmaxf(bf16_lo(m2), bf16_hi(m2));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // 2^(14 - exponent), within the normal numbers
    const int field = min(268 - (int)(__float_as_uint(m) >> 23), 254);
    const float up = __uint_as_float((uint32_t)field << 23), undo = __uint_as_float((uint32_t)(254 - field) << 23);
#pragma unroll
    for (int i = 0; i < kKS; ++i) {
      qf[r][i][0] = pack_f16(bf16_lo(w[2 * i]) * up, bf16_hi(w[2 * i]) * up);
      qf[r][i][1] = pack_f16(bf16_lo(w[2 * i + 1]) * up, bf16_hi(w[2 * i + 1]) * up);
    }
    factor[r][0] = __shfl_sync(0xffffffffu, undo, 8 * c) * P.scale_log2;
    factor[r][1] = __shfl_sync(0xffffffffu, undo, 8 * c + 4) * P.scale_log2;
    lse_add[r] = 0.f;
    if (A.lse != nullptr && A.k_offset != nullptr && split == 0) {        // scores of the keys with their offset: scale q . offset more
      const __nv_bfloat16* const off = (const __nv_bfloat16*)A.k_offset + (int64_t)h * A.D + c * (D / 4);
      float s = 0.f;
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
      lse_add[r] = s * A.sm_scale;
    }
  }
  int limit[NB][2];                        // keys that rows 2 c, 2 c + 1 see
#pragma unroll
  for (int r = 0; r < NB; ++r)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = row0 + r * 8 + 2 * c + j;
      limit[r][j] = row < rows ? seq.seen(A, row / P.group) : 0;
    }

  float o[kKS][NB][4];
  float m_row[NB][2], l_row[NB][2];
#pragma unroll
  for (int r = 0; r < NB; ++r) {
#pragma unroll
    for (int i = 0; i < kKS; ++i) o[i][r][0] = o[i][r][1] = o[i][r][2] = o[i][r][3] = 0.f;
    m_row[r][0] = m_row[r][1] = -INFINITY;
    l_row[r][0] = l_row[r][1] = 0.f;
  }

#pragma unroll 1
  for (int i = 0; i < chunks; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();                          // every lane's part of chunk i is here, and chunk i - 1 has been read by all
    const uint32_t gone = absent >> 2 * (i % kStages) & 3u;
    fetch(i + kStages - 1);
    const uint32_t st = ring + (i % kStages) * kStageBytes;
    const int key0 = begin + kChunk * (kWarps * i + warp);

    float s[kRecs][NB][4];
#pragma unroll
    for (int g = 0; g < kRecs; ++g) {
      const uint32_t rec = st + g * Rec::kBytes;
#pragma unroll
      for (int r = 0; r < NB; ++r) s[g][r][0] = s[g][r][1] = s[g][r][2] = s[g][r][3] = 0.f;
      uint32_t ka[D / 32], kb[D / 32], sa[2], sb[2];            // codes and scales of tokens n, n + 8
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
          mma_f16(s[g][r], x[0], y[0], x[1], y[1], qf[r][2 * w][0], qf[r][2 * w][1]);
          mma_f16(s[g][r], x[2], y[2], x[3], y[3], qf[r][2 * w + 1][0], qf[r][2 * w + 1][1]);
        }
      }
    }

    uint32_t vsc[kRecs];                   // E4M3 of block n (n / 2) and tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
    for (int g = 0; g < kRecs; ++g)
      vsc[g] = lds32(st + g * Rec::kBytes + Rec::kValueScales + (D == 128 ? lane * 4 : (lane >> 3) * 16 + c * 4));

#pragma unroll
    for (int g = 0; g < kRecs; ++g)
#pragma unroll
      for (int r = 0; r < NB; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[g][r][j] *= factor[r][j & 1];
    if (key0 + kChunk > see_all || gone != 0) {
#pragma unroll
      for (int g = 0; g < kRecs; ++g) {
        // Values that no row sees add nothing, whatever lies there.  A NaN scale among the values (E4M3 has no other such code) must
        // not reach rows that do not see its key, so it goes by way of the scores of those that do.
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

    // ---- maxima, P
    uint32_t p[kRecs][NB][2];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      float top[2], corr[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float m = m_row[r][j];
#pragma unroll
        for (int g = 0; g < kRecs; ++g) m = fmaxf(m, fmaxf(s[g][r][j], s[g][r][j + 2]));
        top[j] = m;
      }
#pragma unroll
      for (int d = 4; d < 32; d *= 2) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
      }
      if (__any_sync(0xffffffffu, top[0] > m_row[r][0] || top[1] > m_row[r][1])) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          corr[j] = m_row[r][j] == -INFINITY ? 0.f : ex2_approx(m_row[r][j] - top[j]);
          m_row[r][j] = top[j];
          l_row[r][j] *= corr[j];
        }
#pragma unroll
        for (int i2 = 0; i2 < kKS; ++i2) {
          o[i2][r][0] *= corr[0]; o[i2][r][1] *= corr[1]; o[i2][r][2] *= corr[0]; o[i2][r][3] *= corr[1];
        }
      }
      const float base0 = m_row[r][0] == -INFINITY ? 0.f : m_row[r][0] - kTop, base1 = m_row[r][1] == -INFINITY ? 0.f : m_row[r][1] - kTop;
#pragma unroll
      for (int g = 0; g < kRecs; ++g) {
        const float p0 = ex2_approx(s[g][r][0] - base0), p1 = ex2_approx(s[g][r][1] - base1);
        const float p2 = ex2_approx(s[g][r][2] - base0), p3 = ex2_approx(s[g][r][3] - base1);
        l_row[r][0] += p0 + p2;
        l_row[r][1] += p1 + p3;
        p[g][r][0] = transpose8x8(pack_f16(p0, p1));
        p[g][r][1] = transpose8x8(pack_f16(p2, p3));
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

  // ---- join the four warps
  __syncthreads();
  float* const o_s = reinterpret_cast<float*>(sm);                        // [warp][row][D + 4]
  float2* const ml_s = reinterpret_cast<float2*>(sm + kWarps * kRows * (D + 4) * 4);
  __shared__ float add_s[kRows];
#pragma unroll
  for (int r = 0; r < NB; ++r) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float l = l_row[r][j];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
      const int row = r * 8 + 2 * c + j;
      float* const dst = o_s + (warp * kRows + row) * (D + 4) + n * (D / 8);
#pragma unroll
      for (int i = 0; i < kKS; i += 2)
        *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[i][r][j], o[i][r][2 + j], o[i + 1][r][j], o[i + 1][r][2 + j]);
      if (n == 0) ml_s[warp * kRows + row] = make_float2(m_row[r][j], l);
    }
    if (warp == 0 && c == 0) add_s[r * 8 + n] = lse_add[r];
  }
  __syncthreads();
  constexpr int kPer = kRows * D / (kWarps * 32);                         // channels of a row per thread: 8 (4) or 16 (8)
  const int row = threadIdx.x / (D / kPer), ch = threadIdx.x % (D / kPer) * kPer;
  if (row0 + row >= rows) return;
  float m = -INFINITY, l = 0.f, wgt[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml_s[w * kRows + row].x);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float2 x = ml_s[w * kRows + row];
    wgt[w] = x.x == -INFINITY ? 0.f : ex2_approx(x.x - m);
    l += x.x == -INFINITY ? x.y : wgt[w] * x.y;                           // (a sum of NaN shows although no maximum was found)
  }
  float acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = fmaf(wgt[w], o_s[(w * kRows + row) * (D + 4) + ch + i], acc[i]);
  if (P.splits > 1) {
    const int64_t at = (((int64_t)bh * P.tiles + tile) * P.splits + split) * kRows + row;
#pragma unroll
    for (int i = 0; i < kPer; i += 4)
      *reinterpret_cast<float4*>(P.o_part + at * D + ch + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
    if (ch == 0) P.ml_part[at] = make_float2(m, l);
    if (ch == 0 && split == 0 && A.lse != nullptr) {                      // the joining kernel adds to it
      const int tok = (row0 + row) / P.group, hq = h * P.group + row0 + row - tok * P.group;
      A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = add_s[row];
    }
    return;
  }
  const int tok = (row0 + row) / P.group, hq = h * P.group + row0 + row - tok * P.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh;
#pragma unroll
  for (int i = 0; i < kPer; i += 4)
    if (ch + i < A.D)
      *reinterpret_cast<uint2*>(out + ch + i) = make_uint2(pack_bf16(acc[i] * inv, acc[i + 1] * inv), pack_bf16(acc[i + 2] * inv, acc[i + 3] * inv));
  if (ch == 0 && A.lse != nullptr)
    A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = l == 0.f ? -INFINITY : (m - kTop + log2f(l)) * 0.6931471805599453f + add_s[row];
}

// The ranges of keys of a row joined: a warp per row, a lane D / 32 channels.
template <int D>
__global__ void __launch_bounds__(128) kv_join_kernel(const Params P) {
  const KvAttnArgs& A = P.a;
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int row_id = (int)(id % P.rows_per_tile);
  const int tile = (int)(id / P.rows_per_tile % P.tiles);
  const int64_t bh = id / P.rows_per_tile / P.tiles;
  if (bh >= (int64_t)A.B * A.Hkv) return;                       // (a whole warp; others of the CTA wait below)
  const int b = (int)(bh / A.Hkv), h = (int)(bh - (int64_t)b * A.Hkv);
  const Seq seq(A, b);
  const int rows = seq.q_len * P.group, row = tile * P.rows_per_tile + row_id;
  const int last_row = min(rows, (tile + 1) * P.rows_per_tile) - 1;
  const int used = (seq.seen(A, last_row / P.group) + P.split_keys - 1) / P.split_keys;      // ranges that were written
  pdl_wait();                              // also where there is no row: what follows on the stream may write the first kernel's inputs
  if (row >= rows) return;
  const int64_t at = (bh * P.tiles + tile) * P.splits * P.rows_per_tile + row_id;
  float m = -INFINITY;
  for (int s = lane; s < used; s += 32) m = fmaxf(m, P.ml_part[at + (int64_t)s * P.rows_per_tile].x);
#pragma unroll
  for (int d = 16; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  constexpr int V = D / 32;
  float acc[V], l = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const int64_t x = at + (int64_t)s * P.rows_per_tile;
    const float2 ml = P.ml_part[x];
    const float w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - m);
    l += ml.x == -INFINITY ? ml.y : w * ml.y;
    if constexpr (V == 4) {
      const float4 v = *reinterpret_cast<const float4*>(P.o_part + x * D + lane * 4);
      acc[0] = fmaf(w, v.x, acc[0]); acc[1] = fmaf(w, v.y, acc[1]); acc[2] = fmaf(w, v.z, acc[2]); acc[3] = fmaf(w, v.w, acc[3]);
    } else {
      const float2 v = *reinterpret_cast<const float2*>(P.o_part + x * D + lane * 2);
      acc[0] = fmaf(w, v.x, acc[0]); acc[1] = fmaf(w, v.y, acc[1]);
    }
  }
  const int tok = row / P.group, hq = h * P.group + row - tok * P.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh + lane * V;
  if (lane * V < A.D) {
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16(acc[i] * inv, acc[i + 1] * inv);
  }
  if (lane == 0 && A.lse != nullptr) {
    float* const lse = A.lse + (int64_t)(seq.q0 + tok) * A.Hq + hq;
    *lse = l == 0.f ? -INFINITY : (m - kTop + log2f(l)) * 0.6931471805599453f + (used > 0 ? *lse : 0.f);
  }
}

struct Plan {
  int nb, tiles, splits, split_keys;
};

// 16 rows at a time where there are more than 8; ranges of keys so that the chip is filled about twice.
Plan plan(int B, int Hq, int Hkv, int max_q, int max_k, int sms) {
  Plan p;
  const int64_t rows = (int64_t)max_q * (Hq / Hkv);
  p.nb = rows <= 8 ? 1 : 2;
  p.tiles = (int)((rows + 8 * p.nb - 1) / (8 * p.nb));
  const int64_t ctas = (int64_t)B * Hkv * p.tiles, want = 8 * (int64_t)sms;
  int64_t splits = (want + ctas - 1) / ctas;
  const int64_t most = ((int64_t)max_k + 255) / 256;
  splits = splits < most ? splits : most;
  if (splits < 1) splits = 1;
  const int64_t unit = kWarps * kChunk;
  p.split_keys = (int)(((max_k + splits - 1) / splits + unit - 1) / unit * unit);
  if (p.split_keys < unit) p.split_keys = unit;
  p.splits = (int)(((int64_t)max_k + p.split_keys - 1) / p.split_keys);
  if (p.splits < 1) p.splits = 1;
  return p;
}

template <int D, int NB>
cudaError_t launch(const Params& P, cudaStream_t stream) {
  constexpr int smem = smem_bytes<D, NB>();
  if (cudaError_t e = cudaFuncSetAttribute(kv_decode_kernel<D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); e != cudaSuccess) return e;
  const dim3 grid(P.a.B * P.a.Hkv, P.tiles, P.splits);
  if (cudaError_t e = launch_pdl(kv_decode_kernel<D, NB>, grid, kWarps * 32, smem, stream, false, P); e != cudaSuccess) return e;
  if (P.splits == 1) return cudaGetLastError();
  const int64_t warps = (int64_t)P.a.B * P.a.Hkv * P.tiles * P.rows_per_tile;
  return launch_pdl(kv_join_kernel<D>, dim3((unsigned)((warps + 3) / 4)), 128, 0, stream, true, P);
}

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace

size_t kv_attn_workspace(int B, int Hq, int Hkv, int DS, int max_q, int max_k, int sms) {
  const Plan p = plan(B, Hq, Hkv, max_q, max_k, sms);
  if (p.splits == 1) return 256;
  const size_t rows = (size_t)B * Hkv * p.tiles * p.splits * 8 * p.nb;
  return align256(rows * DS * 4) + align256(rows * 8);
}

cudaError_t launch_kv_attn(const KvAttnArgs& a, cudaStream_t stream) {
  int sms;
  if (cudaError_t e = sm_count(&sms); e != cudaSuccess) return e;
  const Plan p = plan(a.B, a.Hq, a.Hkv, a.max_q, a.max_k, sms);
  if (p.tiles > 65535 || p.splits > 65535) return cudaErrorInvalidValue;
  Params P;
  P.a = a;
  P.group = a.Hq / a.Hkv; P.rows_per_tile = 8 * p.nb; P.tiles = p.tiles; P.splits = p.splits; P.split_keys = p.split_keys;
  P.scale_log2 = a.sm_scale * kLog2e;
  P.page_shift = 0;
  while ((1 << P.page_shift) < a.page_size) ++P.page_shift;
  const size_t rows = (size_t)a.B * a.Hkv * p.tiles * p.splits * 8 * p.nb;
  P.o_part = (float*)a.workspace;
  P.ml_part = (float2*)((char*)a.workspace + align256(rows * a.DS * 4));
  if (a.DS == 128) return p.nb == 1 ? launch<128, 1>(P, stream) : launch<128, 2>(P, stream);
  return p.nb == 1 ? launch<64, 1>(P, stream) : launch<64, 2>(P, stream);
}

}  // namespace sage3
