// What happens to the tokens of a step before attention over the 4-bit cache: block tables and slots, norm and rotation of queries
// and keys, writing keys and values to the cache, and reading them back.
#include "kernels.h"
#include "kv_cache.cuh"

namespace sage3 {

// ------------------------------------------------------------------------------------------------
// Block tables.  With have = ceil(before / ps), need = ceil((before + new) / ps) - have and their exclusive sums, new page number e of
// the step belongs to the request that a search in the sums finds, and so does token t.  One launch: every CTA scans all requests
// (8 bytes each, from L2) into shared memory and then takes its share of pages and tokens, so that one request with a long
// prompt costs no more than many with short ones.  Bound by its latencies, a chain of loads, barriers and searches, and by divisions by the page
// size, four for every request, page and token: 48 requests of one token 3.0 us, 700 requests and 1e5 tokens 8.7 us.
// ------------------------------------------------------------------------------------------------
constexpr int kTableThreads = 256;

// the last i with start[i] <= x, for start[0] = 0 <= x < start[n]
__device__ __forceinline__ int find_owner(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// sum of two counts, held below 2^31 (still associative, so the prefix sums stay sorted whatever the lengths)
__device__ __forceinline__ int add_sat(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }

__global__ void __launch_bounds__(kTableThreads) block_tables_kernel(const KvTablesArgs A) {
  extern __shared__ int sm[];
  int* const cu = sm;                     // tokens before request i
  int* const pages = sm + A.B + 1;        // new pages before request i
  __shared__ int2 warp_sum[kTableThreads / 32];
  const int t = threadIdx.x, per = (A.B + kTableThreads - 1) / kTableThreads;
  const int first = min(t * per, A.B), last = min(first + per, A.B);
  auto lengths = [&](int i, int& before, int& fresh, int& have, int& need) {
    before = max(__ldg(A.before + i), 0);
    fresh = min(max(__ldg(A.fresh + i), 0), 0x7fffffff - before);
    have = (int)(((int64_t)before + A.page_size - 1) / A.page_size);
    need = (int)(((int64_t)before + fresh + A.page_size - 1) / A.page_size) - have;
  };
  int tokens = 0, wanted = 0, before, fresh, have, need;
  for (int i = first; i < last; ++i) {
    lengths(i, before, fresh, have, need);
    tokens = add_sat(tokens, fresh); wanted = add_sat(wanted, need);
  }
  int2 incl = make_int2(tokens, wanted);
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, incl.x, d), y = __shfl_up_sync(0xffffffffu, incl.y, d);
    if ((t & 31) >= d) { incl.x = add_sat(incl.x, x); incl.y = add_sat(incl.y, y); }
  }
  if ((t & 31) == 31) warp_sum[t >> 5] = incl;
  __syncthreads();
  int2 run = make_int2(__shfl_up_sync(0xffffffffu, incl.x, 1), __shfl_up_sync(0xffffffffu, incl.y, 1));
  if ((t & 31) == 0) run = make_int2(0, 0);
  for (int w = 0; w < (t >> 5); ++w) { run.x = add_sat(run.x, warp_sum[w].x); run.y = add_sat(run.y, warp_sum[w].y); }
  for (int i = first; i < last; ++i) {
    lengths(i, before, fresh, have, need);
    cu[i] = run.x; pages[i] = run.y;
    run.x = add_sat(run.x, fresh); run.y = add_sat(run.y, need);
    if (blockIdx.x == 0) A.kv_lens[i] = before + fresh;
  }
  if (t == kTableThreads - 1) {           // (the last thread's range ends at B, or is empty there)
    cu[A.B] = run.x; pages[A.B] = run.y;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = t; i <= A.B; i += kTableThreads) A.cu[i] = cu[i];
    if (t == 0) A.taken[0] = pages[A.B];
  }
  const int at = blockIdx.x * kTableThreads + t, step = gridDim.x * kTableThreads;
  // (Indexes are held to their arrays from both sides: lengths that another stream writes meanwhile may differ between the passes.)
  // New entries; the tokens below take those from the free list too, so nobody reads what is written here
  for (int64_t e = at; e < pages[A.B]; e += step) {
    const int i = find_owner(pages, A.B, (int)e);
    lengths(i, before, fresh, have, need);
    const int64_t col = have + e - pages[i];
    if ((uint64_t)col < (uint64_t)A.cols) A.table[i * A.table_stride + col] = e < A.num_free ? __ldg(A.free_pages + e) : -1;
  }
  for (int64_t x = at; x < A.num_tokens; x += step) {
    int64_t slot = -1;
    int pos = 0;
    if (x < cu[A.B]) {
      const int i = find_owner(cu, A.B, (int)x);
      lengths(i, before, fresh, have, need);
      pos = (int)(before + x - cu[i]);
      const int col = pos / A.page_size;
      int page = -1;
      if ((uint32_t)col < (uint32_t)A.cols) {
        const int64_t e = (int64_t)pages[i] + col - have;
        if (col < have) page = A.table[i * A.table_stride + col];
        else if ((uint64_t)e < (uint64_t)A.num_free) page = __ldg(A.free_pages + e);
      }
      if (page >= 0) slot = (int64_t)page * A.page_size + pos % A.page_size;
    }
    A.positions[x] = pos;
    A.slots[x] = slot;
  }
}

cudaError_t launch_block_tables(const KvTablesArgs& a, cudaStream_t stream) {
  int sms;
  if (cudaError_t e = sm_count(&sms); e != cudaSuccess) return e;
  // The most that any call needs, whatever this one does: what a kernel may use belongs to the kernel, and a call with fewer requests must not
  // take it from one that another thread is about to launch.  (Above 48 KB less the kernel's own 64 bytes it has to be asked for.)
  static std::atomic<uint64_t> allowed;
  if (cudaError_t e = allow_smem(block_tables_kernel, 2 * (kTableMost + 1) * (int)sizeof(int), allowed); e != cudaSuccess) return e;
  const int smem = 2 * (a.B + 1) * (int)sizeof(int);
  const int64_t work = (int64_t)a.num_tokens > a.B ? a.num_tokens : a.B;
  const int ctas = (int)((work + kTableThreads - 1) / kTableThreads);
  block_tables_kernel<<<ctas < sms ? ctas : sms, kTableThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------
// Norm, rotation, cache.  One pass: a lane has 8 channels (16 bytes) of a row, 8 or 16 lanes a row (stored head dim 64 or 128).  A warp
// takes a token's heads `span` at a time, kRows of them loaded before the first is used.
//   y = x rsqrt(mean(x^2) + eps) w,   out = y cos - y' sin  or  y cos + y' sin,   y' the partner's (i +- R/2, or the neighbour i ^ 1)
// What depends on the channel and the token alone, w cos and the partner's w sin, is worked out once for all heads, so a channel costs a
// product, a fused one and the row's factor (520 instructions for 8 rows of 128, half of what it was; N32760, 40 heads of 128 in q and k 412
// -> 227 us, 5.9 TB/s, neighbours paired; halves 240).  All in fp32, one rounding to bf16.  To the cache goes the bf16 value, so that the fused and the separate form store the same bits: x = bf16(k - offset), scale =
// e4m3(max|x| / 6) over the two lanes of a block, code = e2m1(x / scale).  Bound by DRAM.
// Rows whose squares leave fp32's range (channels from 1.6e18 on, below 1e-18 with no eps) are not normed as they should be.  Taking such rows
// again in other units was right and cost every call: N32760, 40 heads 235 -> 263 us with a vote per pass, 286 with a branch per row.
// ------------------------------------------------------------------------------------------------
constexpr int kTokenThreads = 256;

// Codes of 8 channels, inv = 1 / scale.  x / scale is worked out as x * inv, rounded to fp16: x has 8 significant bits and a border between
// codes times the scale 7, so a quotient that is no border is 2^-8 from it, and one that is comes out as the border itself (in fp32
// alone some would miss it by a last bit, 18.75 / 15 for one, and round to the other side).
__device__ __forceinline__ uint32_t quant_codes(const uint4& x, float inv) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  const float2 inv2 = make_float2(inv, inv);
  float2 f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = mul2_ftz(bf16x2_to_f32(w[i]), inv2);
    f[i] = f16x2_to_f32(pack_f16(y.x, y.y));
  }
  return f32x8_to_e2m1x8(f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y);
}
// A block's largest channel, of which a NaN anywhere in the block makes a NaN: its scale then is the NaN of E4M3, and so is all that is read back.
// (The conversion to codes has no NaN and would leave a plausible number.)  Per half of the words max(|a|, |b|); the sign is of no meaning.
__device__ __forceinline__ uint32_t nan_habsmax2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t nan_habsmax2(const uint4& x) { return nan_habsmax2(nan_habsmax2(x.x, x.y), nan_habsmax2(x.z, x.w)); }
__device__ __forceinline__ float nan_absmax(uint32_t x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(bf16_lo(abs2(x))), "f"(bf16_hi(abs2(x))));
  return r;
}
// Codes and scale (of a block of 16 channels, whose other half the next lane has)
__device__ __forceinline__ void quant_half_block(const uint4& x, uint32_t& codes, uint32_t& scale) {
  const uint32_t m2 = nan_habsmax2(x);
  float inv;
  block_scale(nan_absmax(nan_habsmax2(m2, __shfl_xor_sync(0xffffffffu, m2, 1))), scale, inv);     // (its approximate operations are exact on bf16: tests/golden/device_tables)
  codes = quant_codes(x, inv);
}

template <int DS>                         // stored head dim: 64 or 128
__global__ void __launch_bounds__(kTokenThreads, 4) kv_tokens_kernel(const KvTokensArgs A) {
  using Rec = KvRecord<DS>;
  constexpr int kLanes = DS / 8, kPerPass = 32 / kLanes, kPasses = 4, kRows = kPerPass * kPasses;
  const int lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
  const int token = blockIdx.x * (kTokenThreads / 32) + (threadIdx.x >> 5);
  if (token >= A.B * A.N) return;
  const int gq = (A.Hq + A.span - 1) / A.span, gk = (A.Hkv + A.span - 1) / A.span;
  const int g = blockIdx.y, what = g < gq ? 0 : g < gq + gk ? 1 : 2;                 // q, k, v
  const int heads = what == 0 ? A.Hq : A.Hkv, h0 = (what == 0 ? g : what == 1 ? g - gq : g - gq - gk) * A.span, h1 = min(h0 + A.span, heads);
  const int b = A.B == 1 ? 0 : token / A.N, n = token - b * A.N;
  const KvRows& in = what == 0 ? A.q : what == 1 ? A.k : A.vr;
  const bool have = l * 8 < A.D;                                // stored channels beyond the head dim are zero
  const __nv_bfloat16* const src = (const __nv_bfloat16*)in.ptr + b * in.sb + n * in.sn + l * 8;
  const bool to_cache = what != 0 && A.data != nullptr;
  int64_t slot = -1;
  if (to_cache) {
    slot = __ldg(A.slots + token);
    if (slot < 0 || slot >= A.num_slots) slot = -1;
  }

  // ---- the first rows on their way, beside what they are multiplied by
  const __nv_bfloat16* from = src + (h0 + sub) * in.sh;
  const int64_t from_step = kPerPass * in.sh;
  uint4 x[kPasses];
  auto load = [&](int first) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      x[p] = make_uint4(0, 0, 0, 0);
      if (have && first + p * kPerPass + sub < h1) x[p] = *reinterpret_cast<const uint4*>(from);      // (no __ldg: outputs may be the inputs)
      from += from_step;
    }
  };
  load(h0);

  // ---- what the channels of this token are multiplied by: themselves (own), and their partners (other)
  const bool normed = what != 2 && A.weight[what] != nullptr, turned = what != 2 && l * 8 < A.rot, change = what != 2 && (normed || A.rot > 0);
  const int quads = A.rot / 8;                                  // groups of 4 channels in half of the rotated ones
  const bool halves = what != 2 && A.rot > 0 && !A.adjacent;
  float own[8], other[8];
  int src_lane[2] = {lane, lane};                               // of the partners of group 2 l + s of 4 channels (halves)
#pragma unroll
  for (int i = 0; i < 8; ++i) { own[i] = 1.f; other[i] = 0.f; }
  if (change) {
    const __nv_bfloat16* const weight = (const __nv_bfloat16*)A.weight[what];
    float w[8], pw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pw[i] = 1.f;
    if (normed && have) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(weight + l * 8));
      w[0] = bf16_lo(u.x); w[1] = bf16_hi(u.x); w[2] = bf16_lo(u.y); w[3] = bf16_hi(u.y);
      w[4] = bf16_lo(u.z); w[5] = bf16_hi(u.z); w[6] = bf16_lo(u.w); w[7] = bf16_hi(u.w);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) own[i] = w[i];
    if (turned) {
      int64_t place = n;
      if (A.positions != nullptr) place = A.positions64 ? __ldg((const int64_t*)A.positions + token) : (int64_t)__ldg((const int*)A.positions + token);
      const bool known = place >= 0 && place < A.places;        // outside the table: NaN, so that it shows
      const int half = A.rot / 2;
      const float *const cos = A.cos + place * half, *const sin = A.sin + place * half;
      if (A.adjacent) {                                         // pairs (8 l + 2 i, + 1): one angle for two channels
        float4 c4 = make_float4(NAN, NAN, NAN, NAN), s4 = c4;
        if (known) {
          c4 = __ldg(reinterpret_cast<const float4*>(cos + l * 4));
          s4 = __ldg(reinterpret_cast<const float4*>(sin + l * 4));
        }
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          own[2 * i] = w[2 * i] * c[i]; own[2 * i + 1] = w[2 * i + 1] * c[i];
          other[2 * i] = -w[2 * i + 1] * s[i]; other[2 * i + 1] = w[2 * i] * s[i];
        }
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int u = 2 * l + s, pu = u >= quads ? u - quads : u + quads, angle = u >= quads ? pu : u;
          float4 c4 = make_float4(NAN, NAN, NAN, NAN), s4 = c4;
          if (known) {
            c4 = __ldg(reinterpret_cast<const float4*>(cos + angle * 4));
            s4 = __ldg(reinterpret_cast<const float4*>(sin + angle * 4));
          }
          src_lane[s] = lane - l + (pu >> 1);
          if (normed) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(weight + pu * 4));
            pw[4 * s] = bf16_lo(v.x); pw[4 * s + 1] = bf16_hi(v.x); pw[4 * s + 2] = bf16_lo(v.y); pw[4 * s + 3] = bf16_hi(v.y);
          }
          const float c[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w}, sign = u >= quads ? 1.f : -1.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            own[4 * s + i] = w[4 * s + i] * c[i];
            other[4 * s + i] = sign * pw[4 * s + i] * sn[i];
          }
        }
      }
    }
  }

  const KvRows& out = what == 0 ? A.q_out : A.k_out;
  const bool writes = what != 2 && out.ptr != nullptr && have;
  const int64_t page = slot >> A.page_shift;
  const int in_page = (int)slot & (A.page_size - 1), t = in_page & 15;
  const int head_bytes = A.page_size / 16 * Rec::kBytes;
  uint8_t* const base = A.data + page * A.Hkv * head_bytes + in_page / 16 * Rec::kBytes;
  const int code_at = what == 1 ? Rec::key(t, l * 8) : Rec::value(t, l * 8), scale_at = what == 1 ? Rec::key_scale(t, l >> 1) : Rec::value_scale(t, l >> 1);

  const int64_t to_step = kPerPass * out.sh;
  __nv_bfloat16* to = writes ? (__nv_bfloat16*)out.ptr + b * out.sb + n * out.sn + (h0 + sub) * out.sh + l * 8 : nullptr;
#pragma unroll 1
  for (int first = h0; first < h1; first += kRows) {
    if (first != h0) load(first);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int h = first + p * kPerPass + sub;
      if (change) {
        float2 f[4] = {bf16x2_to_f32(x[p].x), bf16x2_to_f32(x[p].y), bf16x2_to_f32(x[p].z), bf16x2_to_f32(x[p].w)};
        float2 o[4];
        if (halves) {
          // the partner's raw words; with an odd number of quads its other half is meant
          uint32_t a0 = x[p].x, a1 = x[p].y, b0 = x[p].z, b1 = x[p].w;
          if (quads & 1) { a0 = x[p].z; a1 = x[p].w; b0 = x[p].x; b1 = x[p].y; }
          o[0] = bf16x2_to_f32(__shfl_sync(0xffffffffu, a0, src_lane[0])); o[1] = bf16x2_to_f32(__shfl_sync(0xffffffffu, a1, src_lane[0]));
          o[2] = bf16x2_to_f32(__shfl_sync(0xffffffffu, b0, src_lane[1])); o[3] = bf16x2_to_f32(__shfl_sync(0xffffffffu, b1, src_lane[1]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = make_float2(f[i].y, f[i].x);
        }
        float r = 1.f;
        if (normed) {
          float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) s2 = ffma2(f[i], f[i], s2);
          float s = s2.x + s2.y;
#pragma unroll
          for (int d = 1; d < kLanes; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
          r = rsqrtf(fmaf(s, A.inv_d, A.eps));
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = f[i].x * own[2 * i];
          y[2 * i + 1] = f[i].y * own[2 * i + 1];
        }
        if (turned) {                      // (elsewhere an infinite neighbour times 0 would be NaN)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = fmaf(o[i].x, other[2 * i], y[2 * i]);
            y[2 * i + 1] = fmaf(o[i].y, other[2 * i + 1], y[2 * i + 1]);
          }
        }
        x[p] = make_uint4(pack_bf16(y[0] * r, y[1] * r), pack_bf16(y[2] * r, y[3] * r), pack_bf16(y[4] * r, y[5] * r), pack_bf16(y[6] * r, y[7] * r));
      }
      if (writes) {
        if (h < h1) *reinterpret_cast<uint4*>(to) = x[p];
        to += to_step;
      }
      if (to_cache) {
        uint4 w = x[p];
        if (what == 1 && A.k_offset != nullptr && have && h < h1)
          w = subtract_mean(w, __ldg(reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.k_offset + h * A.D + l * 8)));
        uint32_t codes, scale;
        quant_half_block(w, codes, scale);
        if (h < h1 && slot >= 0) {
          uint8_t* const rec = base + (int64_t)h * head_bytes;
          *reinterpret_cast<uint32_t*>(rec + code_at) = codes;
          if ((l & 1) == 0) rec[scale_at] = (uint8_t)scale;
        }
      }
    }
  }
}

cudaError_t launch_kv_tokens(KvTokensArgs a, cudaStream_t stream) {
  int sms;
  if (cudaError_t e = sm_count(&sms); e != cudaSuccess) return e;
  const int rows = a.DS == 128 ? 8 : 16;                        // kRows
  const int most = a.Hq > a.Hkv ? a.Hq : a.Hkv, tokens = a.B * a.N;
  // as many heads per warp as leave a round of warps, for which the angles and weights of a token are then fetched once (2000 tokens, 32 + 8
  // heads of 128: two rounds 11.7 us, one 10.6, half a one 12.0)
  const int64_t want = 32ll * sms;
  a.span = rows;
  while (a.span < most && (int64_t)tokens * ((a.Hq + 2 * a.span - 1) / (2 * a.span) + (a.Hkv + 2 * a.span - 1) / (2 * a.span)) >= want) a.span *= 2;
  const int groups = (a.Hq + a.span - 1) / a.span + (a.Hkv + a.span - 1) / a.span * (a.v != nullptr ? 2 : 1);
  if (groups > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)(((int64_t)tokens + kTokenThreads / 32 - 1) / (kTokenThreads / 32)), groups);
  if (a.DS == 128) kv_tokens_kernel<128><<<grid, kTokenThreads, 0, stream>>>(a);
  else kv_tokens_kernel<64><<<grid, kTokenThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------
// Keys and values as they are into the cache, and back.  A thread has a whole block of 16 channels, a warp 4 (8) tokens next to one
// another of a head: their values' codes lie in the same 32-byte sectors.  Blocks a thread has alone need no exchange, and a scale is
// worked out once for 16 channels (20011 tokens, 8 heads of 128, repeated with the writes in L2: 16.7 us against 31 with 8 channels a lane as above, back
// 20.5 against 25; with the writes going out 19.6 and 23.1).
// Slots outside the cache are skipped, and give zeros.
// ------------------------------------------------------------------------------------------------
struct Place {
  uint8_t* rec;
  int t;
};
template <int DS>
__device__ __forceinline__ Place place_of(uint8_t* data, int64_t slot, int page_shift, int heads, int h) {
  const int record = (int)slot & ((1 << page_shift) - 1);
  return Place{data + ((((slot >> page_shift) * heads + h) << (page_shift - 4)) + (record >> 4)) * KvRecord<DS>::kBytes, record & 15};
}

template <int DS>
__global__ void __launch_bounds__(kTokenThreads) kv_append_kernel(const KvTokensArgs A) {
  using Rec = KvRecord<DS>;
  constexpr int kBlocks = DS / 16;
  const int blk = threadIdx.x % kBlocks, token = blockIdx.x * (kTokenThreads / kBlocks) + threadIdx.x / kBlocks, h = blockIdx.y;
  if (token >= A.N) return;
  const int64_t slot = __ldg(A.slots + token);
  const uint4* const src_k = reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.k.ptr + token * A.k.sn + h * A.k.sh) + 2 * blk;
  const uint4* const src_v = reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.vr.ptr + token * A.vr.sn + h * A.vr.sh) + 2 * blk;
  uint4 x[2][2];                          // [k, v]; channels beyond the head dim, a multiple of 8, are zeros
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[0][i] = x[1][i] = make_uint4(0, 0, 0, 0);
    if (blk * 16 + i * 8 < A.D) { x[0][i] = __ldg(src_k + i); x[1][i] = __ldg(src_v + i); }
  }
  if (A.k_offset != nullptr) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (blk * 16 + i * 8 < A.D)
        x[0][i] = subtract_mean(x[0][i], __ldg(reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.k_offset + h * A.D) + 2 * blk + i));
  }
  if (slot < 0 || slot >= A.num_slots) return;
  const Place p = place_of<DS>(A.data, slot, A.page_shift, A.Hkv, h);
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const uint4 u = x[what][0], v = x[what][1];
    uint32_t scale;
    float inv;
    block_scale(nan_absmax(nan_habsmax2(nan_habsmax2(u), nan_habsmax2(v))), scale, inv);
    const uint2 codes = make_uint2(quant_codes(u, inv), quant_codes(v, inv));
    if (what == 0) {
      *reinterpret_cast<uint2*>(p.rec + Rec::key(p.t, blk * 16)) = codes;
      p.rec[Rec::key_scale(p.t, blk)] = (uint8_t)scale;
    } else {
      if (DS == 128) {
        *reinterpret_cast<uint2*>(p.rec + Rec::value(p.t, blk * 16)) = codes;
      } else {                            // (D=64: the values' two groups of 8 channels lie apart)
        *reinterpret_cast<uint32_t*>(p.rec + Rec::value(p.t, blk * 16)) = codes.x;
        *reinterpret_cast<uint32_t*>(p.rec + Rec::value(p.t, blk * 16 + 8)) = codes.y;
      }
      p.rec[Rec::value_scale(p.t, blk)] = (uint8_t)scale;
    }
  }
}

// code times scale is exact in bf16; a key plus its offset is rounded once.  Threads next to one another exchange halves, so that each store
// fills whole 32-byte sectors (with 16 bytes every 32 the L2 took three times the writes).
template <int DS>
__global__ void __launch_bounds__(kTokenThreads) kv_read_kernel(const KvReadArgs A) {
  using Rec = KvRecord<DS>;
  constexpr int kBlocks = DS / 16;
  const int blk = threadIdx.x % kBlocks, token = blockIdx.x * (kTokenThreads / kBlocks) + threadIdx.x / kBlocks, h = blockIdx.y;
  const int64_t slot = token < A.T ? __ldg(A.slots + token) : -1;
  const bool there = slot >= 0 && slot < A.num_slots;
  uint2 codes[2] = {make_uint2(0, 0), make_uint2(0, 0)};       // [k, v]
  uint32_t scale[2] = {0, 0};
  if (there) {
    const Place p = place_of<DS>(const_cast<uint8_t*>(A.data), slot, A.page_shift, A.Hkv, h);
    codes[0] = *reinterpret_cast<const uint2*>(p.rec + Rec::key(p.t, blk * 16));
    scale[0] = p.rec[Rec::key_scale(p.t, blk)];
    if (DS == 128) {
      codes[1] = *reinterpret_cast<const uint2*>(p.rec + Rec::value(p.t, blk * 16));
    } else {
      codes[1].x = *reinterpret_cast<const uint32_t*>(p.rec + Rec::value(p.t, blk * 16));
      codes[1].y = *reinterpret_cast<const uint32_t*>(p.rec + Rec::value(p.t, blk * 16 + 8));
    }
    scale[1] = p.rec[Rec::value_scale(p.t, blk)];
  }
  const bool odd = threadIdx.x & 1;
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const float sf = e4m3_to_f32(scale[what]);
    uint4 y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint4 off = make_uint4(0, 0, 0, 0);
      if (what == 0 && there && A.k_offset != nullptr && blk * 16 + i * 8 < A.D)
        off = __ldg(reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.k_offset + h * A.D + blk * 16) + i);
      uint32_t f[4];
      e2m1x8_to_f16(i == 0 ? codes[what].x : codes[what].y, f);
      const uint32_t o[4] = {off.x, off.y, off.z, off.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = pack_bf16(ffma2(f16x2_to_f32(f[j]), make_float2(sf, sf), bf16x2_to_f32(o[j])));
      y[i] = make_uint4(f[0], f[1], f[2], f[3]);
    }
    // even: its first half and its neighbour's first half; odd: the second halves
    uint4 give = odd ? y[0] : y[1];
    give.x = __shfl_xor_sync(0xffffffffu, give.x, 1); give.y = __shfl_xor_sync(0xffffffffu, give.y, 1);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, 1); give.w = __shfl_xor_sync(0xffffffffu, give.w, 1);
    if (token >= A.T) continue;
    const int ch = (blk & ~1) * 16 + (odd ? 8 : 0);            // of the even block
    uint4* const dst = reinterpret_cast<uint4*>((__nv_bfloat16*)(what == 0 ? A.k : A.v) + ((int64_t)token * A.Hkv + h) * A.D + ch);
    if (ch < A.D) dst[0] = odd ? give : y[0];
    if (ch + 16 < A.D) dst[2] = odd ? y[1] : give;
  }
}

cudaError_t launch_kv_append(const KvTokensArgs& a, cudaStream_t stream) {
  if (a.Hkv > 65535) return cudaErrorInvalidValue;
  const int per = kTokenThreads / (a.DS / 16);
  const dim3 grid((unsigned)((a.N + per - 1) / per), a.Hkv);
  if (a.DS == 128) kv_append_kernel<128><<<grid, kTokenThreads, 0, stream>>>(a);
  else kv_append_kernel<64><<<grid, kTokenThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream) {
  if (a.Hkv > 65535) return cudaErrorInvalidValue;
  const int per = kTokenThreads / (a.DS / 16);
  const dim3 grid((unsigned)((a.T + per - 1) / per), a.Hkv);
  if (a.DS == 128) kv_read_kernel<128><<<grid, kTokenThreads, 0, stream>>>(a);
  else kv_read_kernel<64><<<grid, kTokenThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace sage3
