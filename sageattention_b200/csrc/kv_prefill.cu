// Attention of many query rows per kv head over the 4-bit cache: chunks of prompts behind cached prefixes.
//
// A CTA takes 256 rows (tokens times the heads of a kv head, two tiles of 128) of a (sequence, kv head) and walks tiles of 128 keys:
//   warp  13     fetches a tile's records by bulk copies
//   warps 8-11   turn codes and scales into fp16 (exact, see kv_decode.cu), once for all 256 rows, and write K and V to shared memory.  Both
//                lie alike, rows of keys with 128-byte swizzle: K is then the K-major B operand of S = Q K^T and V the MN-major one
//                of O += P V, so nothing is transposed
//   warp  12     issues the tcgen05.mma kind::f16: S_t = Q_t K^T (queries from shared memory), O_t += P_t V (P from tensor memory)
//   warps 0-3    softmax of row tile 0, a thread per row: scores from tensor memory to registers, weights back to it in fp16
//   warps 4-7    the same for row tile 1; one tile's softmax runs beside the other's MMAs
// Scores are copied whole before they are worked on, which frees their place: a tile's next ones are issued in front of its P V and are there
// when its softmax comes for them.  A row's maximum need not be its maximum (kv_attn.cuh): a thread takes the weights of 128 keys
// against the one that it has, and only where their sum shows one too large for fp16 does it look for the maximum, rescale its
// row of O and take them again.  Weights are rounded to fp16 (by 2^-11 at most) for the MMA, their sum is of what they were.
// The items of the last round have their keys split over CTAs as well and joined by a second kernel.
//
// What bounds it: the instructions of the two softmaxes and of the conversion, which share the SM's four issue ports (the tensor pipe is half
// idle).  Two sequences of 2048 tokens behind 16384 keys, 32 heads of 8, D=128: 862 us, 1196 TFLOP/s of the 1688 that bf16 GEMMs reach; a
// plain form with mma.sync took 5 ms.
//
// Tensor memory (512 columns): O0 [0, D), O1 [D, 2 D), S from 2 D on (128 columns; D=64: two of them), P0 [384, 448), P1 [448, 512).
//
// Every wait on an mbarrier is bounded; where one gives up the CTA records its code in *status, waits (bounded) for its MMAs and copies in
// flight, frees its tensor memory and returns: 60 K stage free, 61 V stage free, 62 Q there, 63 K there, 64 V there, 65 P there, 66 scores
// there, 67 last P V done, 69 records there, 70 scores copied, 71 records read; 68 tensor memory begins elsewhere.
#include "kv_attn.cuh"

namespace sage3 {

namespace {

constexpr int kThreads2 = 512, kM = 128, kN = 128, kItemRows = 2 * kM;
// Register hand-over (setmaxnreg) moves registers inside the pool the CTA was launched with, 128 a thread; launch() checks that.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 192, kFillRegs = 80, kRoleRegs = 48;
static_assert(256 * kSoftmaxRegs + 128 * (kFillRegs + kRoleRegs) <= kThreads2 * kLaunchRegs, "setmaxnreg split exceeds the CTA's register pool");

template <int v>
struct Int {
  static constexpr int value = v;
};

template <int D>
struct Lay {                              // shared memory
  static constexpr int kOperand = kM * D * 2, kHalf = kM * 128;      // a tile; its part of 64 channels
  static constexpr int q = 0, k = 2 * kOperand, v = 4 * kOperand;
  static constexpr int raw = 6 * kOperand, kRaw = kN / 16 * 18 * D;  // a tile's records as they are
  static constexpr int bars = raw + kRaw, total = bars + 256;
  // 16 bytes: channels 8 chunk ... of a row
  static __device__ __forceinline__ int at(int row, int chunk) { return (chunk >> 3) * kHalf + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }
};
struct Bar {                              // byte offsets in the barrier block, of two each but for the last
  static constexpr int k_full = 0, k_empty = 16, v_full = 32, v_empty = 48, q_full = 64, s_full = 80, s_free = 96, p_full = 112, pv_done = 128, drain = 160, raw_full = 168, raw_empty = 176, tmem = 184, abort = 192, there = 196;
};

struct Params2 {
  KvAttnArgs a;
  int group, tiles, page_shift;
  int whole, rest, splits;                // items that a CTA has alone, and those behind them, whose keys are split
  float scale_log2;
  int* status;
  float* o_part;                          // [split, rest, 256, DS]
  float2* ml_part;                        // [split, rest, 256]: maximum (log2) and sum
  float* lse_add;                         // [rest, 256]
};

// Key tiles that the two row tiles of an item see, and a split's share of them
struct Range {
  int n[2], first, count[2];
  __device__ __forceinline__ Range(const KvSeq& seq, const Params2& P, int row0, int rows, int split, int splits) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r0 = row0 + t * kM;
      n[t] = r0 < rows ? (seq.seen(P.a, (min(rows, r0 + kM) - 1) / P.group) + kN - 1) / kN : 0;
    }
    const int all = max(n[0], n[1]), per = (all + splits - 1) / splits;
    first = min(split * per, all);
#pragma unroll
    for (int t = 0; t < 2; ++t) count[t] = max(0, min(min(first + per, all), n[t]) - first);
  }
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 da, {%1, %3};\nmov.b64 db, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 db, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}" ::"r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, const uint32_t (&x)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr) : "memory");
}
// A load's registers may be read once tcgen05.wait::ld is behind it.  Naming them here, behind the wait, ties their readers to it: to the compiler
// they are written by the load, and nothing else keeps a reader from being moved in front of the wait.
template <int N>
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 16)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]),
                      "+r"(r[i + 8]), "+r"(r[i + 9]), "+r"(r[i + 10]), "+r"(r[i + 11]), "+r"(r[i + 12]), "+r"(r[i + 13]), "+r"(r[i + 14]), "+r"(r[i + 15]));
}
// fp16 x fp16 -> fp32, A K-major, B K-major or (transposed) MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int N, bool b_mn) { return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kM >> 4) << 24); }

// What the scales of a lane's values (block n, tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9 of a record of which `seen` keys are seen by any row)
// are replaced by, and whether keys n (bit 0) and n + 8 (bit 1) are to become NaN.  Values of keys that no row sees are zeros, whatever
// lies there.  A NaN scale of a value must not reach rows that do not see its key (0 times NaN): the key becomes NaN in its place,
// whose scores are masked in those rows, and the value 0.
__device__ __noinline__ uint2 mend_scales(uint32_t scales, int seen) {
  const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
  uint32_t nan_keys[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (2 * c + (i & 1) + (i >> 1) * 8 >= seen) scales &= ~(0xffu << (8 * i));
    const bool bad = (scales >> (8 * i) & 0x7fu) == 0x7fu;
    nan_keys[i] = __ballot_sync(0xffffffffu, bad) & (0x11111111u << (n >> 1));
    if (bad) scales &= ~(0xffu << (8 * i));
  }
  return make_uint2(scales, ((n & 1 ? nan_keys[1] : nan_keys[0]) != 0 ? 1u : 0u) | ((n & 1 ? nan_keys[3] : nan_keys[2]) != 0 ? 2u : 0u));
}

template <int D>
__global__ void __launch_bounds__(kThreads2, 1) kv_prefill_kernel(const Params2 P) {
  using Rec = KvRecord<D>;
  using L = Lay<D>;
  constexpr int kSBufs = D == 64 ? 2 : 1;
  constexpr uint32_t kTmS = 2 * D, kTmP = 384;
  extern __shared__ uint8_t raw[];
  const KvAttnArgs& A = P.a;
  uint8_t* const smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const uint32_t base = smem_u32(smem), bars = base + L::bars;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  volatile int* const abort_s = reinterpret_cast<volatile int*>(smem + L::bars + Bar::abort);
  pdl_launch_dependents();

  // ---- the item: the last rows, which see the most keys, first
  const int behind = (int)blockIdx.x - P.whole, splits = behind < 0 ? 1 : P.splits, split = behind < 0 ? 0 : behind / P.rest;
  const int item = behind < 0 ? (int)blockIdx.x : P.whole + behind - split * P.rest;
  const int heads = A.B * A.Hkv, bh = item % heads, tile = P.tiles - 1 - item / heads;
  const int b = bh / A.Hkv, h = bh - b * A.Hkv;
  const KvSeq seq(A, b);
  const int rows = seq.q_len * P.group, row0 = tile * kItemRows;
  const Range R(seq, P, row0, rows, split, splits);
  const int steps = max(R.count[0], R.count[1]);
  // no rows, or no keys among a split's (the joining kernel knows); as one, whatever a warp has read of lengths that another stream writes meanwhile
  if (!__syncthreads_and(row0 < rows && (steps > 0 || splits == 1))) return;
  const int see_any = seq.seen(A, (min(rows, row0 + kItemRows) - 1) / P.group);
  const int* const table = A.table + b * A.table_stride;
  const int key_begin = R.first * kN, key_end = min((R.first + steps) * kN, see_any);
  auto has_page = [&](int key) { return (uint32_t)__ldg(table + (key >> P.page_shift)) < (uint64_t)A.num_pages; };
  int absent = 0;
  for (int key = key_begin + (int)threadIdx.x * A.page_size; key < key_end; key += kThreads2 * A.page_size) absent |= !has_page(key);

  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + Bar::k_full + 8 * i, 4);
      mbar_init(bars + Bar::k_empty + 8 * i, 1);
      mbar_init(bars + Bar::v_full + 8 * i, 4);
      mbar_init(bars + Bar::v_empty + 8 * i, 1);
      mbar_init(bars + Bar::q_full + 8 * i, 4);
      mbar_init(bars + Bar::s_full + 8 * i, 1);
      mbar_init(bars + Bar::s_free + 8 * i, 4);
      mbar_init(bars + Bar::p_full + 8 * i, 4);
      mbar_init(bars + Bar::pv_done + 8 * i, 1);
    }
    mbar_init(bars + Bar::drain, 1);
    mbar_init(bars + Bar::raw_full, 1);
    mbar_init(bars + Bar::raw_empty, 4);
    *abort_s = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(bars + Bar::tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  absent = __syncthreads_or(absent);
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::bars + Bar::tmem);
  int fail = 0;

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
    if (warp == 12) {
      // ---------------------------------------------------------------- MMA
      constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);                     // 8-row groups, version, 128-byte swizzle
      constexpr uint32_t idesc_s = idesc_f16(kN, false), idesc_o = idesc_f16(D, true);
      const uint32_t q_lo = ((base + L::q) >> 4) | (1u << 16), k_lo = ((base + L::k) >> 4) | (1u << 16);
      const uint32_t v_lo = ((base + L::v) >> 4) | ((uint32_t)(L::kHalf >> 4) << 16);     // leading offset: the next 64 channels
      const int count0 = R.count[0], count1 = R.count[1];
      int taken = 0;                       // score tiles issued
      // S of row tile t and key tile j, as soon as the scores that were in its place have been copied; K's stage is free behind the last
      auto scores = [&](int t, int j) {
        if (fail != 0) return;
        const int before = kSBufs == 1 ? taken : j, buf = kSBufs == 1 ? 0 : t;
        if (before > 0 && (fail = wait_bar<70>(bars + Bar::s_free + 8 * buf, (before - 1) & 1)) != 0) return;
        if ((fail = wait_bar<63>(bars + Bar::k_full + 8 * (j & 1), (j >> 1) & 1)) != 0) return;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t a_lo = q_lo + t * (L::kOperand >> 4), b_lo = k_lo + (j & 1) * (L::kOperand >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * L::kHalf + (kk & 3) * 32) >> 4;
            mma_f16_ss(kTmS + buf * kN, a_lo + off, b_lo + off, HI, idesc_s, kk > 0);
          }
          tc_commit(bars + Bar::s_full + 8 * t);
          if (t == 1 || j >= count1) tc_commit(bars + Bar::k_empty + 8 * (j & 1));
        }
        __syncwarp();
        ++taken;
      };
      auto values = [&](int t, int j) {
        if (fail != 0) return;
        if ((fail = wait_bar<64>(bars + Bar::v_full + 8 * (j & 1), (j >> 1) & 1)) != 0) return;
        if ((fail = wait_bar<65>(bars + Bar::p_full + 8 * t, j & 1)) != 0) return;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t b_lo = v_lo + (j & 1) * (L::kOperand >> 4);
#pragma unroll
          for (int kk = 0; kk < kN / 16; ++kk)
            mma_f16_ts(t * D, kTmP + t * 64 + kk * 8, b_lo + kk * (2048 >> 4), HI, idesc_o, kk > 0 ? 1u : j > 0);
          tc_commit(bars + Bar::pv_done + 8 * t);
          if (t == 1 || j >= count1) tc_commit(bars + Bar::v_empty + 8 * (j & 1));
        }
        __syncwarp();
      };
      if (tmem != 0) fail = 68;            // (all of it is this CTA's)
      if (fail == 0 && count0 > 0) fail = wait_bar<62>(bars + Bar::q_full, 0);
      if (fail == 0 && count1 > 0) fail = wait_bar<62>(bars + Bar::q_full + 8, 0);
      // tiles in turn, each one's next scores in front of its P V, so that they are there when its softmax comes for them
      if (count0 > 0) scores(0, 0);
      if (count1 > 0) scores(1, 0);
#pragma unroll 1
      for (int j = 0; j < steps && fail == 0; ++j) {
        if (j + 1 < count0) scores(0, j + 1);
        if (j < count0) values(0, j);
        if (j + 1 < count1) scores(1, j + 1);
        if (j < count1) values(1, j);
      }
      if (fail != 0) {
        give_up(abort_s, P.status, fail);
        if (elect_one()) tc_commit(bars + Bar::drain);
        __syncwarp();
        mbar_wait<true>(bars + Bar::drain, 0, 1u << 16);
      }
    }
    else if (warp == 13) {
      // ---------------------------------------------------------------- records, by bulk copies; which there are goes along
      volatile uint32_t* const there_s = reinterpret_cast<volatile uint32_t*>(smem + L::bars + Bar::there);
      const int64_t page_bytes = (int64_t)A.Hkv * (A.page_size / 16) * Rec::kBytes;
      const uint8_t* const head = A.data + (int64_t)h * (A.page_size / 16) * Rec::kBytes;
      auto page_of = [&](int j) {          // of record `lane` of tile j; -1: no page, or no key that is seen
        const int key = key_begin + j * kN + 16 * lane;
        if (lane >= kN / 16 || key >= key_end) return -1;
        const int page = __ldg(table + (key >> P.page_shift));
        return (uint32_t)page < (uint64_t)A.num_pages ? page : -1;
      };
      int page = steps > 0 ? page_of(0) : -1;
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        if (j > 0 && (fail = wait_bar<71>(bars + Bar::raw_empty, (j - 1) & 1)) != 0) break;
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) {
          *there_s = there;
          mbar_arrive_expect_tx(bars + Bar::raw_full, __popc(there) * Rec::kBytes);
        }
        __syncwarp();
        const int key = key_begin + j * kN + 16 * lane;
        if (page >= 0)
          bulk_load(base + L::raw + lane * Rec::kBytes, head + page * page_bytes + ((key & (A.page_size - 1)) >> 4) * Rec::kBytes, Rec::kBytes, bars + Bar::raw_full);
        __syncwarp();
        page = j + 1 < steps ? page_of(j + 1) : -1;
      }
      if (fail != 0) {
        give_up(abort_s, P.status, fail);
        for (int x = 0; x < 2; ++x) mbar_wait<true>(bars + Bar::raw_full, x, 1u << 16);     // its copies in flight: one of the two phases is past
      }
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- cache -> fp16 tiles: a warp 32 keys of each
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFillRegs));
    const int w = warp & 3, n = lane >> 2, c = lane & 3;
    const uint32_t raw_at = base + L::raw + 2 * w * Rec::kBytes;
    const volatile uint32_t* const there_s = reinterpret_cast<const volatile uint32_t*>(smem + L::bars + Bar::there);
    constexpr int W = D / 32;                                  // words of a lane's codes of a token (keys), of two tokens (values)
    // D=128: half of the lanes take the halves of their 16 bytes in the other order, so that 8 lanes' stores meet different banks.  Keys:
    // rows n, n + 1 and channels 32 c ... fall on the same 128 bytes for c and c + 2.  Values: blocks n and n + 1 do.
    const bool turn_k = D == 128 && c >= 2, turn_v = D == 128 && (n & 1);
    const uint32_t scales_at = raw_at + Rec::kValueScales + (D == 128 ? lane * 4 : (lane >> 3) * 16 + c * 4);
    auto codes = [&](uint32_t at, bool turn, uint32_t (&x)[W]) {
      if constexpr (D == 128) {
        const uint2 u = lds64(at + lane * 16 + (turn ? 8 : 0)), v = lds64(at + lane * 16 + (turn ? 0 : 8));
        x[0] = u.x; x[1] = u.y; x[2] = v.x; x[3] = v.y;
      } else {
        const uint2 u = lds64(at + lane * 8);
        x[0] = u.x; x[1] = u.y;
      }
    };
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      const int stage = j & 1, key0 = key_begin + j * kN + w * 32;
      // two records to registers, so that the next can come
      if ((fail = wait_bar<69>(bars + Bar::raw_full, j & 1)) != 0) break;
      const uint32_t there = *there_s >> (2 * w);
      uint32_t kx[2][2][W], vx[2][2][W], ks[2], vsc[2], poison[2] = {0, 0};
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t rec = raw_at + r * Rec::kBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          codes(rec + i * 4 * D, turn_k, kx[r][i]);
          codes(rec + Rec::kValues + i * 4 * D, turn_v, vx[r][i]);
        }
        vsc[r] = lds32(scales_at + r * Rec::kBytes);
        ks[r] = D == 128 ? lds32(rec + Rec::kKeyScales + lane * 4) : lds16(rec + Rec::kKeyScales + lane * 2);
        if (!(there >> r & 1)) ks[r] = vsc[r] = 0;             // (zeros, then; a page there is not masks its keys as well)
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + Bar::raw_empty);
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (key0 + 16 * r + 16 > see_any || __any_sync(0xffffffffu, (((vsc[r] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0)) {
          const uint2 u = mend_scales(vsc[r], see_any - key0 - 16 * r);
          vsc[r] = u.x; poison[r] = u.y;
        }
      if (j >= 2 && (fail = wait_bar<60>(bars + Bar::k_empty + 8 * stage, ((j >> 1) - 1) & 1)) != 0) break;
      const uint32_t sk = base + L::k + stage * L::kOperand, sv = base + L::v + stage * L::kOperand;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t f0 = e4m3x2_to_f16(ks[r]), f1 = D == 128 ? e4m3x2_to_f16(ks[r] >> 16) : f0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {                          // tokens n, n + 8
          const int row = w * 32 + r * 16 + i * 8 + n;
          uint32_t sc[2];
          if constexpr (D == 128) {
            sc[0] = __byte_perm(i ? f1 : f0, 0, turn_k ? 0x3232 : 0x1010); sc[1] = __byte_perm(i ? f1 : f0, 0, turn_k ? 0x1010 : 0x3232);
          } else {
            sc[0] = sc[1] = __byte_perm(f0, 0, i ? 0x3232 : 0x1010);
          }
          if (poison[r] >> i & 1) sc[0] = sc[1] = 0x7e007e00u;
#pragma unroll
          for (int z = 0; z < W; ++z) {
            uint32_t y[4];
            e2m1x8_to_f16(kx[r][i][z], y);
#pragma unroll
            for (int u = 0; u < 4; ++u) y[u] = hmul2(y[u], sc[D == 128 ? z >> 1 : 0]);
            sts128(sk + L::at(row, c * W + (turn_k ? z ^ 2 : z)), y);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + Bar::k_full + 8 * stage);
      if (j >= 2 && (fail = wait_bar<61>(bars + Bar::v_empty + 8 * stage, ((j >> 1) - 1) & 1)) != 0) break;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) {                          // tokens 2 c + 8 i and the next, or (turn) the other way round
          const uint32_t f = e4m3x2_to_f16(vsc[r] >> (16 * i));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = w * 32 + r * 16 + i * 8 + 2 * c + (turn_v ? e ^ 1 : e);
            const uint32_t sc = __byte_perm(f, 0, (turn_v ? e == 0 : e == 1) ? 0x3232 : 0x1010);
#pragma unroll
            for (int z = 0; z < W / 2; ++z) {
              uint32_t y[4];
              e2m1x8_to_f16(vx[r][i][e * (W / 2) + z], y);
#pragma unroll
              for (int u = 0; u < 4; ++u) y[u] = hmul2(y[u], sc);
              sts128(sv + L::at(row, n * (W / 2) + z), y);
            }
          }
        }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + Bar::v_full + 8 * stage);
    }
    if (fail != 0) give_up(abort_s, P.status, fail);
  } else {
    // ---------------------------------------------------------------- softmax: thread r of the warpgroup has row r of its tile
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2, r = (warp & 3) * 32 + lane, row = row0 + t * kM + r, count = R.count[t];
    const bool real = row < rows;
    const int tok = real ? row / P.group : 0, hq = h * P.group + (real ? row - tok * P.group : 0);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem + kTmS + (kSBufs == 1 ? 0 : t) * kN + lanes, tm_o = tmem + t * D + lanes, tm_p = tmem + kTmP + t * 64 + lanes;
    float factor, add = 0.f;
    {
      const uint4* const src = reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.q + (int64_t)(seq.q0 + tok) * A.q_sn + hq * A.q_sh);
      uint4 x[D / 8];
      uint32_t m2 = 0;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        x[i] = make_uint4(0, 0, 0, 0);
        if (real && i * 8 < A.D) x[i] = __ldg(src + i);
        m2 = habsmax2(m2, habsmax2(habsmax2(x[i].x, x[i].y), habsmax2(x[i].z, x[i].w)));
      }
      m2 = abs2(m2);
      const RowScale scale(fmaxf(bf16_lo(m2), bf16_hi(m2)));
      factor = fmaxf(scale.undo * P.scale_log2, 1.2e-38f);     // (never 0: it multiplies the -inf of masked scores)
      if (A.lse != nullptr && A.k_offset != nullptr && split == 0 && real) {          // scores of the keys with their offset: scale q . offset more
        const uint4* const off = reinterpret_cast<const uint4*>((const __nv_bfloat16*)A.k_offset + (int64_t)h * A.D);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          if (i * 8 < A.D) {
            const uint4 o = __ldg(off + i);
            add = fmaf(bf16_lo(x[i].x), bf16_lo(o.x), fmaf(bf16_hi(x[i].x), bf16_hi(o.x), add));
            add = fmaf(bf16_lo(x[i].y), bf16_lo(o.y), fmaf(bf16_hi(x[i].y), bf16_hi(o.y), add));
            add = fmaf(bf16_lo(x[i].z), bf16_lo(o.z), fmaf(bf16_hi(x[i].z), bf16_hi(o.z), add));
            add = fmaf(bf16_lo(x[i].w), bf16_lo(o.w), fmaf(bf16_hi(x[i].w), bf16_hi(o.w), add));
          }
        add *= A.sm_scale;
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t y[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) y[z] = pack_f16(bf16_lo(u[z]) * scale.up, bf16_hi(u[z]) * scale.up);
        sts128(base + L::q + t * L::kOperand + L::at(r, i), y);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + Bar::q_full + 8 * t);
    }
    const int limit = real ? seq.seen(A, tok) : 0x7fffffff;    // keys that the row sees
    const int limit_all = __reduce_min_sync(0xffffffffu, limit);
    float m = kLowest;
    float2 l = make_float2(0.f, 0.f);
    // One key tile: its scores to registers, so that the next ones can be on their way, then their weights.  Masks stay out of the loop that
    // nearly all tiles take.
    auto key_tile = [&](auto masked_, int j) {
      constexpr bool masked = decltype(masked_)::value != 0;
      if ((fail = wait_bar<66>(bars + Bar::s_full + 8 * t, j & 1)) != 0) return;
      tc_fence_after();
      // (whether P's place is free: a look takes hundreds of cycles beside busy warps, so it lies beside the copy)
      const bool place_free = j == 0 || mbar_test(bars + Bar::pv_done + 8 * t, (j - 1) & 1);
      uint32_t s[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32(tm_s + 32 * i, s[i]);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_loaded(s[i]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + Bar::s_free + 8 * (kSBufs == 1 ? 0 : t));
      if (masked) {
        const int key0 = key_begin + j * kN;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (key0 + 32 * i + x >= limit) s[i][x] = 0xff800000u;
        if (absent) {                      // some page of the item's keys is not in the cache (the whole CTA knows)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (key0 + 16 * i < key_end && !has_page(key0 + 16 * i)) {
#pragma unroll
              for (int x = 0; x < 16; ++x) s[i >> 1][(i & 1) * 16 + x] = 0xff800000u;
            }
        }
      }
      if (!__all_sync(0xffffffffu, place_free) && (fail = wait_bar<67>(bars + Bar::pv_done + 8 * t, (j - 1) & 1)) != 0) return;
      tc_fence_after();
      float2 both;
#pragma unroll 1
      for (bool again = false;; again = true) {
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 f2 = make_float2(factor, factor), base2 = make_float2(kTop - m, kTop - m);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t p[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            float2 e = ffma2(make_float2(__uint_as_float(s[i][2 * x]), __uint_as_float(s[i][2 * x + 1])), f2, base2);
            e.x = ex2_approx(e.x); e.y = ex2_approx(e.y);
            sum[x & 1] = fadd2(sum[x & 1], e);
            p[x] = pack_f16(e.x, e.y);
          }
          tmem_st16(tm_p + 16 * i, p);
        }
        both = fadd2(sum[0], sum[1]);
        // a weight too large for fp16 makes the sum larger than 2^15 (and where it is, one of the 128 is 2^8 at least); so does a NaN
        const bool bad = !(both.x + both.y <= 32768.f) || m == kLowest;
        if (__builtin_expect(again || !__any_sync(0xffffffffu, bad), 1)) break;
        // Once more with the maximum of these scores.  Rows that are well get the same weights again: no row's bits depend on another row.
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 32; x += 2) top = fmaxf(top, fmaxf(__uint_as_float(s[i][x]), __uint_as_float(s[i][x + 1])));
        const float m_new = bad ? fmaxf(m, top * factor) : m, corr = ex2_approx(m - m_new);
        m = m_new;
        l.x *= corr; l.y *= corr;
        if (j > 0) {
#pragma unroll 1
          for (int i = 0; i < D / 16; ++i) {
            uint32_t o[16];
            tmem_ld16(tm_o + 16 * i, o);
            tmem_wait_ld();
            tmem_loaded(o);
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * corr);
            tmem_st16(tm_o + 16 * i, o);
          }
        }
      }
      l = fadd2(l, both);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + Bar::p_full + 8 * t);
    };
    const int plain = absent ? 0 : max(0, min(count, (limit_all - key_begin) / kN));     // tiles all of whose keys every row of the warp sees
    int j = 0;
#pragma unroll 1
    for (; j < plain && fail == 0; ++j) key_tile(Int<0>{}, j);
#pragma unroll 1
    for (; j < count && fail == 0; ++j) key_tile(Int<1>{}, j);
    if (fail == 0 && count > 0) fail = wait_bar<67>(bars + Bar::pv_done + 8 * t, (count - 1) & 1);
    if (fail != 0) {
      give_up(abort_s, P.status, fail);
    } else if (splits == 1 || count > 0) {
      tc_fence_after();
      const float sum = l.x + l.y, inv = sum == 0.f ? 0.f : 1.0f / sum;
      const int64_t place = (int64_t)(item - P.whole) * kItemRows + t * kM + r;          // (where the keys are split)
      const int64_t part = (int64_t)split * P.rest * kItemRows + place;
      __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh;
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        if (count > 0) {
          tmem_ld32(tm_o + 32 * i, o);
          tmem_wait_ld();
          tmem_loaded(o);
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0;
        }
        if (real) {
          if (splits == 1) {
#pragma unroll
            for (int x = 0; x < 32; x += 8)
              if (32 * i + x < A.D) {
                uint32_t y[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) y[z] = pack_bf16(__uint_as_float(o[x + 2 * z]) * inv, __uint_as_float(o[x + 2 * z + 1]) * inv);
                *reinterpret_cast<uint4*>(out + 32 * i + x) = make_uint4(y[0], y[1], y[2], y[3]);
              }
          } else {
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<uint4*>(P.o_part + part * D + 32 * i + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          }
        }
      }
      if (real && splits > 1) P.ml_part[part] = make_float2(m, sum);
      if (real && A.lse != nullptr) {
        if (splits == 1) A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = lse_of(m, sum, add);
        else if (split == 0) P.lse_add[place] = add;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The splits of a row joined: a warp per row, a lane D / 32 channels, in the order of the keys.
template <int D>
__global__ void __launch_bounds__(256) kv_prefill_join_kernel(const Params2 P) {
  constexpr int V = D / 32;
  const KvAttnArgs& A = P.a;
  const int lane = threadIdx.x & 31;
  const uint32_t id = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int in_tile = id % kItemRows, heads = A.B * A.Hkv, item = P.whole + id / kItemRows, bh = item % heads, tile = P.tiles - 1 - item / heads;
  const int b = bh / A.Hkv, h = bh - b * A.Hkv;
  const KvSeq seq(A, b);
  const int rows = seq.q_len * P.group, row = tile * kItemRows + in_tile;
  pdl_wait();                              // also where there is no row: what follows on the stream may write the first kernel's inputs
  if (row >= rows) return;
  const Range R(seq, P, tile * kItemRows, rows, 0, P.splits);
  const int n = R.n[in_tile / kM], all = max(R.n[0], R.n[1]), per = (all + P.splits - 1) / P.splits;
  const int used = n > 0 ? (n + per - 1) / per : 0;
  const int64_t place = id, step = (int64_t)P.rest * kItemRows;
  float m = kLowest;
  for (int s = lane; s < used; s += 32) m = fmaxf(m, P.ml_part[place + s * step].x);
#pragma unroll
  for (int d = 16; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float acc[V], l = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const int64_t at = place + s * step;
    const float2 ml = P.ml_part[at];
    const float w = ex2_approx(ml.x - m);
    l = fmaf(w, ml.y, l);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(P.o_part + at * D + lane * V + i);
      acc[i] = fmaf(w, v.x, acc[i]); acc[i + 1] = fmaf(w, v.y, acc[i + 1]);
    }
  }
  const int tok = row / P.group, hq = h * P.group + row - tok * P.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __nv_bfloat16* const out = (__nv_bfloat16*)A.out + (int64_t)(seq.q0 + tok) * A.o_sn + hq * A.o_sh + lane * V;
  if (lane * V < A.D) {
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16(acc[i] * inv, acc[i + 1] * inv);
  }
  if (lane == 0 && A.lse != nullptr) A.lse[(int64_t)(seq.q0 + tok) * A.Hq + hq] = lse_of(m, l, used > 0 ? P.lse_add[place] : 0.f);
}

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

struct Plan2 {
  int tiles, whole, rest, splits;
  size_t add, ml, o, bytes;               // offsets in the workspace
};

// As many items as there are SMs take as long as one, so those of the last round have their keys split over CTAs, into as many parts as
// make it shortest by this account, in key tiles: what an item costs beside its tiles, the joining, and a sixteenth for each partial result.
// (us, whole items -> so, 32 heads of 8, D=128: B2 1200 tokens 16384 keys 665 -> 526, 2048 tokens 911 -> 862; B1 1600 tokens 8192 keys 213 -> 187.)
constexpr int kItemCost = 6, kJoinCost = 10;

Plan2 plan2(int B, int Hq, int Hkv, int DS, int max_q, int max_k, int sms) {
  Plan2 p;
  p.tiles = (int)(((int64_t)max_q * (Hq / Hkv) + kItemRows - 1) / kItemRows);
  const int items = (int)((int64_t)B * Hkv * p.tiles), key_tiles = (int)(((int64_t)max_k + kN - 1) / kN);
  p.rest = items % sms;
  p.whole = items - p.rest;
  p.splits = 1;
  int64_t best = INT64_MAX;
  for (int n = 1; p.rest > 0 && p.rest * (n - 1) < 4 * sms && 4 * (n - 1) <= key_tiles; ++n) {
    const int rounds = (p.rest * n + sms - 1) / sms, tiles = (key_tiles + n - 1) / n + kItemCost;
    const int64_t cost = 16ll * rounds * tiles + (n > 1 ? 16 * kJoinCost + p.rest * n : 0);
    if (cost < best) { best = cost; p.splits = n; }
  }
  if (p.splits == 1) { p.whole += p.rest; p.rest = 0; }
  const size_t rows = (size_t)p.rest * kItemRows;
  p.add = 256;
  p.ml = p.add + align256(rows * 4);
  p.o = p.ml + align256(rows * p.splits * 8);
  p.bytes = p.o + align256(rows * p.splits * DS * 4);
  return p;
}

template <int D>
cudaError_t launch(const Params2& P, const Plan2& p, cudaStream_t stream) {
  constexpr int smem = Lay<D>::total + 1024;
  // asked once: what the register hand-over relies on
  static const cudaError_t regs_ok = [] {
    cudaFuncAttributes f;
    const cudaError_t e = cudaFuncGetAttributes(&f, kv_prefill_kernel<D>);
    return e != cudaSuccess ? e : f.numRegs < kLaunchRegs ? cudaErrorInvalidConfiguration : cudaSuccess;
  }();
  if (regs_ok != cudaSuccess) return regs_ok;
  static std::atomic<uint64_t> allowed;
  if (cudaError_t e = allow_smem(kv_prefill_kernel<D>, smem, allowed); e != cudaSuccess) return e;
  if (cudaError_t e = launch_pdl(kv_prefill_kernel<D>, dim3((unsigned)(p.whole + p.rest * p.splits)), kThreads2, smem, stream, false, P); e != cudaSuccess) return e;
  if (p.rest == 0) return cudaGetLastError();
  return launch_pdl(kv_prefill_join_kernel<D>, dim3((unsigned)((int64_t)p.rest * kItemRows / 8)), 256, 0, stream, true, P);
}

}  // namespace

// Rows per kv head from which on this kernel takes over.  kv_decode.cu turns a key's codes into fp16 once for 24 (32) rows, this one once
// for 256, but works on 128 rows at least.  Decode / prefill, 32 heads of 8, 4096 keys, us: B16 D=128 24 rows 37.8 / 51.6, 32 rows 51.7 /
// 51.6; D=64 32 rows 31.3 / 46.3, 48 rows 41.2 / 46.3; B4 D=128 24 rows 15.8 / 23.9, 32 rows 24.8 / 23.9.
bool kv_prefill_takes(int Hq, int Hkv, int DS, int max_q) { return (int64_t)max_q * (Hq / Hkv) > (DS == 128 ? 32 : 48); }

size_t kv_prefill_workspace(int B, int Hq, int Hkv, int DS, int max_q, int max_k, int sms) { return plan2(B, Hq, Hkv, DS, max_q, max_k, sms).bytes; }

bool kv_prefill_fits(int B, int Hq, int Hkv, int max_q) {
  const int64_t rows = (int64_t)max_q * (Hq / Hkv), tiles = (rows + kItemRows - 1) / kItemRows;
  return (int64_t)B * Hkv * tiles * kItemRows < (1ll << 31);
}

cudaError_t launch_kv_prefill(const KvAttnArgs& a, cudaStream_t stream) {
  int sms;
  if (cudaError_t e = sm_count(&sms); e != cudaSuccess) return e;
  const Plan2 p = plan2(a.B, a.Hq, a.Hkv, a.DS, a.max_q, a.max_k, sms);
  Params2 P;
  P.a = a;
  P.group = a.Hq / a.Hkv; P.tiles = p.tiles; P.whole = p.whole; P.rest = p.rest; P.splits = p.splits;
  P.scale_log2 = a.sm_scale * kLog2e;
  P.page_shift = 0;
  while ((1 << P.page_shift) < a.page_size) ++P.page_shift;
  char* const w = (char*)a.workspace;
  P.status = a.status != nullptr ? a.status : (int*)w;
  P.lse_add = (float*)(w + p.add); P.ml_part = (float2*)(w + p.ml); P.o_part = (float*)(w + p.o);
  return a.DS == 128 ? launch<128>(P, p, stream) : launch<64>(P, p, stream);
}

}  // namespace sage3
