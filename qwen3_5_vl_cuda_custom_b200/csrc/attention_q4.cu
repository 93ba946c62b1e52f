// Attention over a 4-bit KV cache (layout: kv_q4.cuh).
//
// out[b, s, h D + d] = sum_k p_k V[k, d] / sum_k p_k, p_k = exp(scale q . K[k] - max),
// over the keys k < len_b, with a causal mask aligned to the last key (query s
// of Sq sees k <= s + len_b - Sq).  A row that sees no key is zero.
//
// What bounds it: a key and its value are 160 bytes at D = 128 (groups of 32),
// read once, so a long cache should run at memory speed; but each of those bytes
// is two codes to unpack, so the instructions per code decide.  Per SM and clock
// HBM delivers about 24 bytes = 48 codes against 128 lanes of issue, 64 of them
// for logic operations.
//
// Codes as they stand.  The bits c << 4 (c = 0..15) read as bf16 are c * 2^-129 and the
// bits c are c * 2^-133, as fp16 c * 2^-20 and c * 2^-24: the subnormals and the first
// binade are evenly spaced.  The matrix units and fma.f16x2 take subnormals at full
// precision, so `w & 0x000f000f` and `w & 0x00f000f0` are pairs of codes, without
// a conversion or an offset to take out again; one shift by 8 gives the other
// four codes of a word.  The powers of two go into the other operand.
//
// Scores.  With K = m + s c per group j, q . K = sum_j s_j (Q_j . c_j) + m_j sum(Q_j).
// Q is scaled by 2^X, which brings the largest of a group's queries into [2^60, 2^61)
// (X at most 75, so queries below 2^-15 are left smaller), and by 2^52 (codes at bit 0)
// or 2^48 (at bit 4), so a product is 2^(X-81) Q . c; the minima go through one more
// matrix instruction whose other operand is 2^(X-81) sum(Q_j) split into three bf16 parts
// (24 bits).  So K is never rounded, and the scale costs one fp32 operation per key,
// query and group.  Queries 2^-100 of their group's largest lose bits; |Q| < 2^100.
//
// Keys are the 16 rows of the instruction and queries its 8 columns (S^T = K Q^T,
// O^T = V^T P^T): a decode step has G = Hq/Hkv queries per kv head, often 8, and
// no half of the tile is idle.  P moves from accumulator to operand layout by an
// 8x8 transpose between the lanes (movmatrix).
//
// Values.  P and V go into their product as fp16, of 11 bits: rounded to bf16 each
// would cost as much as the output's own rounding (relative error of normal data
// 0.0022 to 0.0026; 0.0016 like this, which is the output's rounding alone).  For the
// range that bf16 has and fp16 has not, every key has a power of two F: V 2^-F enters,
// dequantised in registers as (2^-24 c) (2^(24-F) s) + 2^-F m (16 times that for the
// codes at bit 4), and the key's weight is 2^F p, by an F added to its score.  So the
// running maximum is that of what the keys contribute, a key with a large V and a small
// weight costs the others nothing, nor does a masked one; the sum of weights takes
// 2^-F out again.  F is the least one at which 2^(24-F) s < 2^16 and 2^(4-F) |m| < 2^15
// for all groups of the key, so V is off by at most 2^-11 of itself or 2^-15 of the
// largest s of its key (a code step is s).  Weights reach 2^15 (kLift), so they have
// all 11 bits down to 2^-29 of the largest.
// Visible values: |V| between 2^-60 and 2^100, rows of 0 counting as 2^-60.  Where two
// visible rows are 2^105 apart the smaller one's weight no longer enters the sum (fp32's
// smallest number is 2^-126, the larger one's weight 2^15): beside zeros, 2^40 is safe.
//
// V's operand wants pairs of neighbouring keys.  A transposing ldmatrix over the
// codes as 16-bit units (four codes) gives exactly that: a lane receives, for two
// keys, the unit of its column, so its eight V channels per 16-byte chunk pair
// come without a byte permutation and belong to one scale group.
//
// Work.  A group is a (sequence, kv head, 8 NT query rows); its 32-key tiles go in
// rounds of four, one tile per warp.  The rounds of all groups form one list, each
// group headed by one more round for what it costs to begin and end it, and the
// list is cut into equal runs, one per resident CTA; a run may end one group, take
// several whole and begin another.  Nothing depends on the lengths being alike,
// and the rings below do not drain between groups.  A group that one run holds
// whole is written at once, the others leave (max, sum, O) partials that a second
// kernel joins; a run leaves at most two.  When there are many short groups, runs are of
// whole groups, and of single warps: a warp takes all tiles of a group one after the
// other, and nothing is joined.
//
// Each warp keeps its tiles coming through a private ring of asynchronous 16-byte
// copies, so warps meet only at the end of a group.  The 16-byte chunks of a row
// are XOR-swizzled by the row, so that both the 16-byte reads of K and the 8-row
// reads of V touch every bank once.
//
// Measured in a captured graph (32/4 heads x 128, groups of 32): 64 sequences x 8193 keys
// 69.2 us, 4.9 TB/s (the copies alone 61; a plain copy moves 6.5 TB/s); one sequence x
// 131072 keys 23.9 us; x 500 keys 7.4 us.  595 warp instructions per 32-key tile, issue
// slots 59 % busy: what bounds it is copies and arithmetic together, the 16x8 matrix
// instructions (one per 2 clocks and SM) holding up the logic operations beside them.
// More than 16 query rows unpack every key again: 64 sequences x 8192 keys, 2 kv heads, 8,
// 16, 32, 64 and 128 rows 41.8, 68.3, 96.9, 250 and 354 us.
// Tried: P and V in bf16 (64.0 us when this form took 68.7, the errors above), P as two
// bf16 parts (70.8, 0.0021 to 0.0023); e4m3 operands for K (emulated: 48M instructions
// for 37M), shifts as multiplications (12 % slower), a tile's scores together with the
// products of the tile before (17 %), bulk copies instead of 16-byte ones.
#include <cuda_fp16.h>
#include <float.h>

#include <type_traits>

#include "kv_q4.cuh"

namespace q35 {
namespace {

using q4::Cache;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;  // keys per tile
// CTAs per SM, and tiles in flight per warp.  At D = 128 the registers allow 3 CTAs with
// 8 query rows and 2 with 16 (64 sequences x 8193 keys: 4 CTAs of 128 registers 73.7 us,
// 3 68.7; 16 rows, 2 kv heads: 3 with spills 94, 2 71); at D = 64 and 32 3 with either
// (16 rows, 2 kv heads: 2 CTAs 54.6 and 45.0 us, 3 38.9 and 29.1).
constexpr int ctas_per_sm(int d, int nt) { return d == 128 && nt == 2 ? 2 : 3; }
constexpr float kLift = 15.f;   // weights reach 2^kLift
constexpr int kMinF = -60;      // smallest F of a key
constexpr int stages(int d, int nt) { return d == 128 && nt == 1 ? 2 : 4; }

struct Params {
  const uint16_t *q;
  Cache c;
  uint16_t *out;
  float *ws;
  const int32_t *kv_lens;
  int *err;
  int B, Hq, Hkv, G, Sq, R, n_rg, causal;
  int runs;   // CTAs of the main kernel
  int per;    // rounds of a run (unless scan)
  int scan;   // runs are cut by the sequences' own lengths (kv_lens)
  int kv_len;
  int64_t cap;
  float scale_log2;
};

template <int D, int GS, int NT>
struct Layout {
  static constexpr int J = D / 32;       // code words per lane and key
  static constexpr int NS = D / GS;      // scale words per key
  static constexpr int kStages = stages(D, NT);
  static constexpr int kCodes = kTile * D / 2, kScales = kTile * NS * 4;
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kRing = kStages * kStage;
  static constexpr int kRegs = NT * (D / 4 + 4);  // a lane's O, m, l
  // (F, 2^-F) of a tile's keys, V's scales and minima as fp16
  static constexpr int kKeys = kTile * (8 + 16 + 16);
  static constexpr int kSmem = kWarps * (kRing + kKeys) + (kWarps - 1) * kRegs * 128;
};

// Workspace: [2 runs][8 NT rows][D] floats and [2 runs][8 NT rows] (m, l) of partials
// (slot 2 r holds the group that run r continues, 2 r + 1 the one it begins), then
// with kv_lens the first round of every sequence and the number of all rounds.
constexpr int64_t partial_rows(int64_t runs, int nt) { return 2 * runs * 8 * nt; }

__device__ __forceinline__ int clamp_len(const Params &p, int b) {
  if (!p.kv_lens) return p.kv_len;
  return max(0, min(p.kv_lens[b], p.kv_len));
}
// Rounds of a group in the list: its tiles by `share`, the warps that take part in it
// (a sequence without rows counts one, so that someone writes its zeros), behind one for
// its start and end.
__host__ __device__ __forceinline__ int rounds_of(int len, int share = kWarps) {
  return 1 + (len > 0 ? (len + share * kTile - 1) / (share * kTile) : 1);
}

// A group of the list: its sequence, its (kv head, row group) index, its first
// round, the sequence's length in keys and rounds.
struct Group {
  int b, hg, begin, len, rounds;
};
// Prefix sums over the sequences' rounds by the whole CTA.  Returns the rounds of
// all groups; finds the sequence that holds round at(total) and sets its first
// round.  `table` (or null) receives every sequence's first round and the total.
template <typename At>
__device__ __forceinline__ int scan_rounds(const Params &p, At &&at, Group &gr, int *table) {
  __shared__ int warp_sum[kWarps], found[2];
  const int tid = threadIdx.x, lane = tid & 31;
  const int each = (p.B + kThreads - 1) / kThreads, b0 = tid * each, b1 = min(b0 + each, p.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += rounds_of(clamp_len(p, b));
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) warp_sum[tid >> 5] = incl;
  __syncthreads();
  int total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < (tid >> 5)) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int unit = p.Hkv * p.n_rg;
  total *= unit;
  const int want = at(total);
  for (int b = b0; b < b1; ++b) {
    const int t = rounds_of(clamp_len(p, b));
    if (want >= before * unit && want - before * unit < t * unit) {
      found[0] = b;
      found[1] = before * unit;
    }
    if (table) table[b] = before * unit;
    before += t;
  }
  if (table && tid == 0) table[p.B] = total;
  __syncthreads();
  gr.b = found[0];
  gr.begin = found[1];
  return total;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
  const int n = live ? 16 : 0;  // 0: the 16 bytes become zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// D = A(16x16) * B(16x8) + C, fp32: bf16 operands, and fp16.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1,
                                    float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The codes of fields 0..3 and 4..7 of a word as 16-bit pairs (field i, field i + 4):
// as bf16 c * 2^-133 for i = 0, 2 and c * 2^-129 for i = 1, 3, as fp16 c * 2^-24 and
// c * 2^-20.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t (&c)[4]) {
  const uint32_t h = w >> 8;
  c[0] = w & 0x000f000fu;
  c[1] = w & 0x00f000f0u;
  c[2] = h & 0x000f000fu;
  c[3] = h & 0x00f000f0u;
}
// fp16 pairs; subnormals count.
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// Larger magnitudes of bf16 pairs (the signs are of no use; a NaN gives way).
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t addr) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}
template <int N>
__device__ __forceinline__ void sts_words(uint32_t addr, const uint32_t (&w)[N]) {
  if constexpr (N == 4)
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};"
                 ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  else if constexpr (N == 2)
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(w[0]), "r"(w[1]) : "memory");
  else
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(w[0]) : "memory");
}
__device__ __forceinline__ uint32_t lds1(uint32_t addr) {
  uint32_t w[1];
  lds_words<1>(w, addr);
  return w[0];
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ bool nonfinite(uint32_t pair) {
  return (((pair & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
}

// One CTA = one run of tiles (SHARE = 4), or each of its warps has one of its own (1).
template <int D, int GS, int NT, int SHARE>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D, NT)) attn_q4_kernel(Params p) {
  using L = Layout<D, GS, NT>;
  constexpr int J = L::J, NS = L::NS, BPG = GS / 32;
  constexpr int RB = D / 2;                     // bytes of a row of codes
  constexpr int CH = RB / 16;                   // 16-byte chunks of it
  constexpr int MT = D / 16;                    // 16-channel tiles of O^T
  extern __shared__ __align__(128) uint8_t smem[];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per_seq = p.Hkv * p.n_rg;
  constexpr bool kAlone = SHARE == 1;
  const int part = kAlone ? 0 : warp;        // the warp's tile of a round
  constexpr int kRound = SHARE * kTile;      // keys of a round

  if (p.kv_lens) wait_for_earlier();
  // ---- the run [lo, hi) of rounds and the group it begins in
  Group gr;
  int lo, hi;
  if (!kAlone && p.scan) {
    int per = 0;
    int *table = reinterpret_cast<int *>(p.ws + partial_rows(p.runs, NT) * (D + 2));
    const int total = scan_rounds(p, [&](int n) {
      per = (n + p.runs - 1) / p.runs;
      return static_cast<int>(min(int64_t(blockIdx.x) * per, int64_t(n)));
    }, gr, blockIdx.x == 0 ? table : nullptr);
    lo = static_cast<int>(min(int64_t(blockIdx.x) * per, int64_t(total)));
    hi = min(lo + per, total);
  } else {
    const int all = rounds_of(p.kv_len, SHARE) * per_seq;
    lo = (kAlone ? blockIdx.x * kWarps + warp : blockIdx.x) * p.per;
    hi = min(lo + p.per, all * p.B);
    gr.b = lo / all;
    gr.begin = gr.b * all;
  }
  if (p.kv_lens && blockIdx.x == 0)
    for (int b = tid; b < p.B; b += kThreads)
      if (p.kv_lens[b] < 0 || p.kv_lens[b] > p.kv_len)
        report_error(p.err, DEV_ERR_INDEX, 311, b, p.kv_lens[b]);
  if (lo >= hi) return;
  auto seq_rounds = [&](int len) { return rounds_of(!kAlone && p.scan ? len : p.kv_len, SHARE); };
  gr.len = clamp_len(p, gr.b);
  gr.rounds = seq_rounds(gr.len);
  gr.hg = (lo - gr.begin) / gr.rounds;
  gr.begin += gr.hg * gr.rounds;
  auto next_group = [&](Group &x) {
    x.begin += x.rounds;
    if (++x.hg == per_seq) {
      x.hg = 0;
      x.len = clamp_len(p, ++x.b);
      x.rounds = seq_rounds(x.len);
    }
  };

  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * L::kRing;
  const uint32_t keys = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) +
                        kWarps * L::kRing + warp * L::kKeys;
  const uint32_t vscale = keys + kTile * 8 + lane * 16;
  float *merge = reinterpret_cast<float *>(smem + kWarps * (L::kRing + L::kKeys));

  // ---- copies: this warp's tiles (tile SHARE r + part of round r of a group), ahead of
  // their use.  Lane i copies chunks i, i + 32, ... of the tile's codes (chunk c of row
  // r goes to chunk c ^ swizzle(r)) and chunk i of its scales.  Rows behind the length
  // are not read (a chunk of narrow scales may hold up to 3 of them: the capacity is a
  // multiple of 16).
  constexpr int kCopies = L::kCodes / 512;  // code copies per lane, of K and of V
  const int crow = lane / CH, cch = lane % CH;
  const int csw = D == 128 ? (crow >> 1) & 3 : D == 64 ? (crow >> 2) & 1 : 0;
  const uint32_t cdst = crow * RB + ((cch ^ csw) << 4);
  const int srow = lane * 4 / NS;           // first row of the lane's chunk of scales
  Group ahead = gr;
  int next = lo, ahead_end = gr.begin + gr.rounds;
  // first row of this warp's tile of round `next` in its group (negative: the mark)
  int r0 = (lo - gr.begin - 1) * kRound + part * kTile;
  const uint8_t *kc_at, *vc_at, *ks_at, *vs_at;  // the group's row 0 (this lane's chunks)
  auto ahead_at = [&]() {
    const int64_t row = (int64_t(ahead.b) * p.Hkv + ahead.hg / p.n_rg) * p.cap;
    kc_at = reinterpret_cast<const uint8_t *>(p.c.k_codes) + row * RB + lane * 16;
    vc_at = reinterpret_cast<const uint8_t *>(p.c.v_codes) + row * RB + lane * 16;
    ks_at = reinterpret_cast<const uint8_t *>(p.c.k_scales) + row * (NS * 4) + lane * 16;
    vs_at = reinterpret_cast<const uint8_t *>(p.c.v_scales) + row * (NS * 4) + lane * 16;
  };
  ahead_at();
  uint32_t next_stage = 0;  // byte offset in the ring
  auto issue = [&]() {
    for (; next < hi; ++next, r0 += kRound) {  // to the next round with a tile for this warp
      if (next >= ahead_end) {
        next_group(ahead);
        ahead_end = ahead.begin + ahead.rounds;
        r0 = part * kTile - kRound;
        ahead_at();
      }
      if (static_cast<uint32_t>(r0) < static_cast<uint32_t>(ahead.len)) break;
    }
    if (next < hi) {
      const int left = ahead.len - r0;
      const uint32_t dst = ring + next_stage;
      const uint8_t *kc = kc_at + int64_t(r0) * RB, *vc = vc_at + int64_t(r0) * RB;
      if (left >= kTile) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          copy16(dst + cdst + i * 512, kc + i * 512, true);
          copy16(dst + L::kCodes + L::kScales + cdst + i * 512, vc + i * 512, true);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const bool live = crow + i * (32 / CH) < left;
          copy16(dst + cdst + i * 512, live ? kc + i * 512 : kc, live);
          copy16(dst + L::kCodes + L::kScales + cdst + i * 512, live ? vc + i * 512 : vc, live);
        }
      }
      if (lane < L::kScales / 16) {
        const int64_t off = int64_t(r0) * (NS * 4);
        const bool live = srow < left;
        copy16(dst + L::kCodes + lane * 16, ks_at + (live ? off : 0), live);
        copy16(dst + 2 * L::kCodes + L::kScales + lane * 16, vs_at + (live ? off : 0), live);
      }
      ++next;
      r0 += kRound;
      next_stage = next_stage + L::kStage == L::kRing ? 0 : next_stage + L::kStage;
    }
    copies_commit();
  };
  if (!p.kv_lens) wait_for_earlier();
  let_next_launch();  // (in front of the wait, several kernels in a row would crowd some SMs)
#pragma unroll 1
  for (int i = 0; i < L::kStages; ++i) issue();

  // Addresses within a stage.  K: 4 J bytes of row g (and g + 8) per lane, words
  // t J .. of it; V: row (lane & 7) of the 8x8 matrix lane / 8.
  const int ksw = D == 128 ? (g >> 1) & 3 : D == 64 ? (g >> 2) & 1 : 0;
  const uint32_t koff = g * RB + (D == 128 ? (t ^ ksw) << 4 : D == 64 ? (((t >> 1) ^ ksw) << 4) + (t & 1) * 8
                                                                    : t * 4);
  // matrices: D >= 64 (chunk pair, key block of 8): chunk m / 2, keys 8 (m & 1); D = 32: keys 8 m
  const int vrow = (lane & 7) + (D == 32 ? lane & 24 : lane & 8);
  const int vsw = D == 128 ? (vrow >> 1) & 3 : D == 64 ? (vrow >> 2) & 1 : 0;
  const int vch = D == 32 ? 0 : lane >> 4;
  const int gv = (D == 128 ? g >> 1 : D == 64 ? (g >> 1) & 1 : 0) / BPG;  // the lane's V scale group
  uint32_t stage = 0;

  for (int at = lo; at < hi;) {
    // ---- one group's part of the run: its rounds [at, end), the first round of the
    // group being only a mark
    const int end = min(hi, gr.begin + gr.rounds);
    const int b = gr.b, hk = gr.hg / p.n_rg, rg = gr.hg - hk * p.n_rg, len = gr.len;
    const bool begins = at <= gr.begin + 1, whole = begins && end == gr.begin + gr.rounds;
    if (end == gr.begin + 1) {
      at = end;
      if (at < hi) next_group(gr);
      continue;
    }

    // Query rows: row r -> head hk G + r / Sq, position r % Sq.  Column g of an
    // operand tile holds 8 channels of every 32; accumulator columns are 2t, 2t + 1.
    uint32_t qf[NT][J][4];
    uint32_t qm[NT][2];  // 2^(X-81) sum(Q_t) of group t in three bf16 parts
    int lim[NT][2];      // keys the column's query sees
    uint32_t largest = 0u;  // exponent
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t top = 0u;
      const int r = (rg * NT + nt) * 8 + g;
      const uint16_t *src = nullptr;
      if (r < p.R) {
        const int h = r / p.Sq, s = r - h * p.Sq;
        src = p.q + ((int64_t(b) * p.Hq + hk * p.G + h) * p.Sq + s) * D;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint4 x = src ? *reinterpret_cast<const uint4 *>(src + 32 * j + 8 * t)
                            : make_uint4(0u, 0u, 0u, 0u);
        qf[nt][j][0] = x.x, qf[nt][j][1] = x.y, qf[nt][j][2] = x.z, qf[nt][j][3] = x.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max_abs2(top, qf[nt][j][i]);
      }
      // (an infinite query spoils its own row; the others' power of two goes by the rest)
      const uint32_t e0 = top >> 7 & 0xffu, e1 = top >> 23 & 0xffu;
      largest = max(largest, max(e0 == 255u ? 0u : e0, e1 == 255u ? 0u : e1));
    }
    const int e = __reduce_max_sync(0xffffffffu, largest);
    const int up_by = max(-60, min(187 - e, 75));  // X
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 52 + up_by) << 23);
    const float scale_up = p.scale_log2 * 0x1p20f *
                           __uint_as_float(static_cast<uint32_t>(127 + 61 - up_by) << 23);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum[NS];
#pragma unroll
      for (int j = 0; j < NS; ++j) sum[j] = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float lo, hi;
          unpack_bf2(qf[nt][j][i], lo, hi);
          sum[j / BPG] += lo + hi;
          const float f = i % 2 == 0 ? up : up * 0x1p-4f;
          qf[nt][j][i] = pack_bf2(lo * f, hi * f);
        }
      }
      float mine = 0.f;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        float v = sum[j];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        if (j == t) mine = v * (up * 0x1p-133f);
      }
      const float h0 = bf2f(f2bf(mine)), h1 = bf2f(f2bf(mine - h0));
      qm[nt][0] = pack_bf2(h0, h1);
      qm[nt][1] = pack_bf2(mine - h0 - h1, 0.f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rc = (rg * NT + nt) * 8 + 2 * t + c;
        lim[nt][c] = p.causal ? min(len, len - p.Sq + rc % p.Sq + 1) : len;
      }
    }
    const int lim_all = p.causal ? min(len, len - p.Sq + 1) : len;  // keys every query sees

    float o[MT][NT][4];
    float row_m[NT][2], row_l[NT][2];  // in units of log2; l of this lane's keys only
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      row_m[nt][0] = row_m[nt][1] = -FLT_MAX;
      row_l[nt][0] = row_l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
    }

    for (int round = max(at, gr.begin + 1); round < end; ++round) {
      const int key0 = (round - gr.begin - 1) * kRound + part * kTile;
      if (key0 >= len) break;
      copies_wait<L::kStages - 1>();
      __syncwarp();
      const uint32_t sk = ring + stage;
      const uint32_t sks = sk + L::kCodes, sv = sks + L::kScales, svs = sv + L::kCodes;

      const bool partial = key0 + kTile > lim_all;
      if (partial) {
        // A weight of 0 does not silence a NaN or an infinity in V: rows behind the
        // length are cleared, and a non-finite group that some query must not see is
        // cleared too and put into the outputs of the queries that do see it.
        const bool behind = key0 + lane >= len;
        uint32_t clear = behind ? (1u << NS) - 1u : 0u;  // groups of key row `lane`
        if (!behind) {
#pragma unroll
          for (int i = 0; i < NS; ++i)
            if (nonfinite(lds1(svs + (lane * NS + i) * 4))) clear |= 1u << i;
        }
        uint32_t todo = __ballot_sync(0xffffffffu, clear != 0 && !behind);
        while (todo) {
          const int kk = __ffs(todo) - 1;
          todo &= todo - 1;
          if (nonfinite(lds1(svs + (kk * NS + gv) * 4))) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (key0 + kk < lim[nt][e & 1]) o[i][nt][e] = NAN;
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (clear >> i & 1u)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(svs + (lane * NS + i) * 4), "r"(0u) : "memory");
        __syncwarp();
      }
      uint32_t vw[NS];  // V's scales and minima of key `lane`
      lds_words<NS>(vw, svs + lane * (NS * 4));

      // ---- S^T = K Q^T (two blocks of 16 keys) + F, in units of log2
      float s[2][NT][4], unf[2][2];  // unf: 2^-F
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t wl[J], wh[J], pl[NS], ph[NS];
        const int kl = 16 * mt + g;
        lds_words<J>(wl, sk + 16 * mt * RB + koff);
        lds_words<J>(wh, sk + (16 * mt + 8) * RB + koff);
        lds_words<NS>(pl, sks + kl * (NS * 4));
        lds_words<NS>(ph, sks + (kl + 8) * (NS * 4));
        // minima: (m, m, m) of group t times the parts of its sum(Q)
        const uint32_t m0 = __byte_perm(lds1(sks + (kl * NS + t % NS) * 4), 0u, 0x3232);
        const uint32_t m1 = __byte_perm(lds1(sks + ((kl + 8) * NS + t % NS) * 4), 0u, 0x3232);
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma(s[mt][nt], m0, m1, m0, m1, qm[nt][0], qm[nt][1], 0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          uint32_t a[4], c[4];
          codes4(wl[j], a);
          codes4(wh[j], c);
          const int sg = j / BPG;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (j % BPG == 0)
              mma(part[nt], a[0], c[0], a[1], c[1], qf[nt][j][0], qf[nt][j][1], 0.f, 0.f, 0.f, 0.f);
            else
              mma(part[nt], a[0], c[0], a[1], c[1], qf[nt][j][0], qf[nt][j][1], part[nt][0],
                  part[nt][1], part[nt][2], part[nt][3]);
            mma(part[nt], a[2], c[2], a[3], c[3], qf[nt][j][2], qf[nt][j][3], part[nt][0],
                part[nt][1], part[nt][2], part[nt][3]);
          }
          if (j % BPG == BPG - 1) {
            const float s0 = __uint_as_float(pl[sg] << 16), s1 = __uint_as_float(ph[sg] << 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              s[mt][nt][0] = fmaf(s0, part[nt][0], s[mt][nt][0]);
              s[mt][nt][1] = fmaf(s0, part[nt][1], s[mt][nt][1]);
              s[mt][nt][2] = fmaf(s1, part[nt][2], s[mt][nt][2]);
              s[mt][nt][3] = fmaf(s1, part[nt][3], s[mt][nt][3]);
            }
          }
        }
        if (mt == 0) {
          // V's scales and minima as fp16, by a power of two 2^-F per key, and F for the
          // key's weights
          uint32_t top = vw[0];
#pragma unroll
          for (int i = 1; i < NS; ++i) top = max_abs2(top, vw[i]);
          const int f = max(kMinF + 127, max(static_cast<int>(top >> 7 & 0xffu) + 9,
                                             static_cast<int>(top >> 23 & 0xffu) - 10));
          const float fs = __uint_as_float((278 - f) << 23), fm = fs * 0x1p-20f;  // 2^(24-F), 2^(4-F)
          // for a transposing ldmatrix: word j of the key's row serves lanes g = 2j, 2j + 1
          uint32_t vs[4], vm[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w = vw[(D == 128 ? j : D == 64 ? j & 1 : 0) / BPG];
            const float sc = __uint_as_float(w << 16) * fs, mi = __uint_as_float(w & 0xffff0000u) * fm;
            vs[j] = pack_h2(sc, sc);
            vm[j] = pack_h2(mi, mi);
          }
          sts_words<4>(vscale, vs);
          sts_words<4>(vscale + kTile * 16, vm);
          const uint32_t k2[2] = {
              __float_as_uint(__uint_as_float(0x4b000000u | f) - (8388608.f + 127.f)),
              __float_as_uint(fs * 0x1p-24f)};
          sts_words<2>(keys + lane * 8, k2);
        }
      }
      __syncwarp();
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t f0[2], f1[2];
        lds_words<2>(f0, keys + (16 * mt + g) * 8);
        lds_words<2>(f1, keys + (16 * mt + g + 8) * 8);
        unf[mt][0] = __uint_as_float(f0[1]);
        unf[mt][1] = __uint_as_float(f1[1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[mt][nt][e] = fmaf(s[mt][nt][e], scale_up, __uint_as_float(e < 2 ? f0[0] : f1[0]));
      }
      if (partial) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + 16 * mt + g + 8 * (e >> 1) >= lim[nt][e & 1]) s[mt][nt][e] = -INFINITY;
      }

      // ---- softmax: the maximum is raised (and O rescaled) only when some key exceeds it
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx0 = fmaxf(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[1][nt][0], s[1][nt][2]));
        float mx1 = fmaxf(fmaxf(s[0][nt][1], s[0][nt][3]), fmaxf(s[1][nt][1], s[1][nt][3]));
        if (__any_sync(0xffffffffu, mx0 > row_m[nt][0] || mx1 > row_m[nt][1])) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
          }
          mx0 = fmaxf(mx0, row_m[nt][0]);
          mx1 = fmaxf(mx1, row_m[nt][1]);
          const float a0 = exp2_fast(row_m[nt][0] - mx0), a1 = exp2_fast(row_m[nt][1] - mx1);
          row_m[nt][0] = mx0;
          row_m[nt][1] = mx1;
          row_l[nt][0] *= a0;
          row_l[nt][1] *= a1;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[i][nt][0] *= a0;
            o[i][nt][1] *= a1;
            o[i][nt][2] *= a0;
            o[i][nt][3] *= a1;
          }
        }
        // rounded up: scores whose fp32 step is above 1 must not lift a weight past fp16
        const float mu0 = __fadd_ru(row_m[nt][0], -kLift), mu1 = __fadd_ru(row_m[nt][1], -kLift);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float p0 = exp2_fast(s[mt][nt][0] - mu0), p1 = exp2_fast(s[mt][nt][1] - mu1);
          const float p2 = exp2_fast(s[mt][nt][2] - mu0), p3 = exp2_fast(s[mt][nt][3] - mu1);
          row_l[nt][0] = fmaf(p2, unf[mt][1], fmaf(p0, unf[mt][0], row_l[nt][0]));
          row_l[nt][1] = fmaf(p3, unf[mt][1], fmaf(p1, unf[mt][0], row_l[nt][1]));
          pb[mt][nt][0] = transpose8x8(pack_h2(p0, p1));
          pb[mt][nt][1] = transpose8x8(pack_h2(p2, p3));
        }
      }

      // ---- O^T += V^T P^T
      uint32_t u[4], vs[4], vm[4];
      ldsm4_t(vs, vscale);
      ldsm4_t(vm, vscale + kTile * 16);
      if constexpr (D == 32) ldsm4_t(u, sv + vrow * RB);  // keys 0-7, 8-15, 16-23, 24-31
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        // scale pairs of keys (2t, 2t + 1) and (2t + 8, 2t + 9); minima for even and odd fields
        const uint32_t s2[2] = {vs[2 * mt], vs[2 * mt + 1]};
        uint32_t m2[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          m2[h][1] = vm[2 * mt + h];
          m2[h][0] = mul2(m2[h][1], 0x2c002c00u);  // 2^-4
        }
        auto product = [&](int tile, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, int i) {
          a0 = fma2(a0, s2[0], m2[0][i]);
          a1 = fma2(a1, s2[0], m2[0][i]);
          a2 = fma2(a2, s2[1], m2[1][i]);
          a3 = fma2(a3, s2[1], m2[1][i]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float(&acc)[4] = o[tile][nt];
            mma_f16(acc, a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
          }
        };
        if constexpr (D == 32) {
          // rows g and g + 8 of tile i: fields i and i + 2 of the lane's unit
          uint32_t x[4], y[4];
          codes4(u[2 * mt], x);
          codes4(u[2 * mt + 1], y);
#pragma unroll
          for (int i = 0; i < 2; ++i) product(i, x[i], x[i + 2], y[i], y[i + 2], i);
        } else {
#pragma unroll
          for (int cp = 0; cp < CH / 2; ++cp) {
            // matrices: (chunk 2cp, keys 0-7), (2cp, 8-15), (2cp + 1, 0-7), (2cp + 1, 8-15);
            // rows g and g + 8 of tile 4 cp + i: field i of the unit in chunks 2cp and 2cp + 1
            ldsm4_t(u, sv + (16 * mt + vrow) * RB + (((2 * cp + vch) ^ vsw) << 4));
            uint32_t x[4], x8[4], y[4], y8[4];
            codes4(u[0], x);
            codes4(u[1], x8);
            codes4(u[2], y);
            codes4(u[3], y8);
#pragma unroll
            for (int i = 0; i < 4; ++i) product(4 * cp + i, x[i], y[i], x8[i], y8[i], i % 2);
          }
        }
      }
      __syncwarp();
      issue();
      stage = stage + L::kStage == L::kRing ? 0 : stage + L::kStage;
    }

    // ---- join the warps (lane i of every warp holds the same rows and channels)
    // and write the group's rows or its partials
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nt][e] *= i % 2 == 0 ? 0x1p-15f : 0x1p-19f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      row_l[nt][0] *= 0x1p-15f;
      row_l[nt][1] *= 0x1p-15f;
    }
    if constexpr (!kAlone) __syncthreads();
    if (part > 0) {
      float *dst = merge + (warp - 1) * (L::kRegs * 32) + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          dst[((D / 4 + 4) * nt + c) * 32] = row_m[nt][c];
          dst[((D / 4 + 4) * nt + 2 + c) * 32] = row_l[nt][c];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[((D / 4 + 4) * nt + 4 + 4 * i + e) * 32] = o[i][nt][e];
      }
    }
    if constexpr (!kAlone) __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float *src = merge + (D / 4 + 4) * nt * 32 + lane;
        float f[SHARE][2], l[2], m[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mw[kWarps - 1];
          m[c] = row_m[nt][c];
#pragma unroll
          for (int w = 0; w < SHARE - 1; ++w) {
            mw[w] = src[(w * L::kRegs + c) * 32];
            m[c] = fmaxf(m[c], mw[w]);
          }
          f[0][c] = kAlone ? 1.f : exp2_fast(row_m[nt][c] - m[c]);
          l[c] = row_l[nt][c] * f[0][c];
#pragma unroll
          for (int w = 0; w < SHARE - 1; ++w) {
            f[w + 1][c] = exp2_fast(mw[w] - m[c]);
            l[c] = fmaf(src[(w * L::kRegs + 2 + c) * 32], f[w + 1][c], l[c]);
          }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], d);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = o[i][nt][e] * f[0][e & 1];
#pragma unroll
            for (int w = 0; w < SHARE - 1; ++w)
              v = fmaf(src[(w * L::kRegs + 4 + 4 * i + e) * 32], f[w + 1][e & 1], v);
            o[i][nt][e] = v;
          }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int lr = nt * 8 + 2 * t + c, r = rg * 8 * NT + lr;
          const bool live = r < p.R;
          const float inv = !whole ? 1.f : l[c] == 0.f ? 0.f : 1.0f / l[c];
          const int h = r / p.Sq, sq = r - h * p.Sq;
          uint16_t *dst = p.out + ((int64_t(b) * p.Sq + sq) * p.Hq + hk * p.G + h) * D;
          const int64_t row = (2 * int64_t(blockIdx.x) + (begins ? 1 : 0)) * (8 * NT) + lr;
          // A unit is channels 32 j + 8 k + 2 i + (g & 1), i = 0..3: lanes g and g ^ 1 hold
          // the even and the odd ones and trade halves, for four neighbours each.
#pragma unroll
          for (int un = 0; un < (D == 32 ? 1 : CH); ++un) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = (D == 32 ? o[i % 2][nt][c + 2 * (i / 2)]
                              : o[4 * (un / 2) + i][nt][c + 2 * (un % 2)]) * inv;
            const bool odd = g & 1;
            const float r0 = __shfl_xor_sync(0xffffffffu, odd ? x[0] : x[2], 4);
            const float r1 = __shfl_xor_sync(0xffffffffu, odd ? x[1] : x[3], 4);
            const float4 v = odd ? make_float4(r0, x[2], r1, x[3]) : make_float4(x[0], r0, x[1], r1);
            const int j = D == 128 ? g >> 1 : D == 64 ? (g >> 1) & 1 : 0;
            const int k = D == 128 ? un : D == 64 ? 2 * un + (g >> 2) : g >> 1;
            const int ch = 32 * j + 8 * k + (odd ? 4 : 0);
            if (live && whole)
              *reinterpret_cast<uint2 *>(dst + ch) = make_uint2(pack_bf2(v.x, v.y), pack_bf2(v.z, v.w));
            if (live && !whole) *reinterpret_cast<float4 *>(p.ws + row * D + ch) = v;
          }
          if (live && !whole && g == 0)
            reinterpret_cast<float2 *>(p.ws + partial_rows(p.runs, NT) * D)[row] =
                make_float2(m[c], l[c]);
        }
      }
    }
    at = end;
    if (at < hi) next_group(gr);
  }
  copies_wait<0>();
}

// One CTA per query row: joins the runs that share the row's group.  Each warp joins
// the partials it loads, U at once, by their own maximum.
template <int D, int WARPS, int U>
__global__ void __launch_bounds__(WARPS * 32) attn_q4_join_kernel(Params p, int rows_per_group) {
  constexpr int E = D / 32;
  __shared__ float part[WARPS][D], part_m[WARPS], part_l[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gr = blockIdx.x, bh = gr / p.R, r = gr - bh * p.R;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int rg = r / rows_per_group, lr = r - rg * rows_per_group;
  wait_for_earlier();
  let_next_launch();
  int per = p.per, begin, rounds;
  if (p.scan) {
    const int *table = reinterpret_cast<const int *>(p.ws + 2 * int64_t(p.runs) * rows_per_group * (D + 2));
    begin = table[b];
    rounds = rounds_of(clamp_len(p, b));
    per = (table[p.B] + p.runs - 1) / p.runs;
  } else {
    rounds = rounds_of(p.kv_len);
    begin = b * p.Hkv * p.n_rg * rounds;
  }
  begin += (hk * p.n_rg + rg) * rounds;
  const int c0 = (begin + 1) / per;  // the run with the group's first keys
  const int n = (begin + rounds - 1) / per - c0 + 1;
  if (n == 1) return;  // one run held the group and wrote the row
  auto slot = [&](int i) {
    return (2 * (int64_t(c0) + i) + (i == 0 ? 1 : 0)) * rows_per_group + lr;
  };
  const float2 *ml = reinterpret_cast<const float2 *>(p.ws + 2 * int64_t(p.runs) * rows_per_group * D);
  float m = -FLT_MAX, l = 0.f, v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
  for (int i0 = warp; i0 < n; i0 += U * WARPS) {
    float x[U][E];
    float2 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * WARPS;
      const int64_t at = slot(i < n ? i : 0);
      w[u] = i < n ? ml[at] : make_float2(-FLT_MAX, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = i < n ? p.ws[at * D + 32 * e + lane] : 0.f;
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, w[u].x);
    const float keep = exp2_fast(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= keep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = exp2_fast(w[u].x - m);
      l = fmaf(w[u].y, f, l);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = fmaf(x[u][e], f, v[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) part[warp][32 * e + lane] = v[e];
  if (lane == 0) {
    part_m[warp] = m;
    part_l[warp] = l;
  }
  __syncthreads();
  for (int d = tid; d < D; d += WARPS * 32) {
    float top = -FLT_MAX, lt = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) top = fmaxf(top, part_m[i]);
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float f = exp2_fast(part_m[i] - top);
      lt = fmaf(part_l[i], f, lt);
      sum = fmaf(part[i][d], f, sum);
    }
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    const int h = r / p.Sq, sq = r - h * p.Sq;
    p.out[((int64_t(b) * p.Sq + sq) * p.Hq + hk * p.G + h) * D + d] = f2bf(sum * inv);
  }
}

// Query rows per CTA, and the runs the rounds are cut into.  All plans go by the
// device's SMs, not by a thread's limit: what the workspace was asked for is what any
// launch of the same sizes takes.
struct Plan {
  int nt, n_rg, runs, per;
  bool scan, join, alone;  // alone: a warp per group
};
// When to cut groups: a round at D = 128 takes about 0.8 us while every CTA has an SM
// to itself and 1.6 once some SMs hold two or three; the second kernel adds 2.2 us and
// 0.025 us per query row, 1.3 more when lengths on the device cut the runs.  That, in
// tenths of a lone round, fits both forms' times at 96 shapes (head_dim 64 and 128, 1 to
// 256 sequences, 128 to 4096 keys; 0.5 % above the better one on average).  Another 1.8
// us is counted because the second launch and its workspace cost the host 4 us, which a
// short call waits for outside a graph (on the device it costs 1 % on average).
// 8 sequences x 4 kv heads: 512 keys whole 6.7, cut 7.1 us; 1024 keys 10.0 and 8.4; 256
// sequences: 1024 keys 46 and 49, 4096 keys 151 and 131.
int round_cost(int64_t ctas, int D) {
  return (ctas <= device_sms() ? 10 : 20) * (D + 192) / 320;
}
int64_t join_cost(int64_t rows, bool lens) { return 50 + rows / 32 + (lens ? 16 : 0); }
// Query rows of a group, in eights.  16 rows unpack a key once for two instructions, but
// a round takes longer and there are fewer: by the rounds of a run, from both forms'
// times at 12 to 64 rows (D = 128, 64, 32; one sequence x 32768 to 64 x 8192 keys).
// 2 kv heads x 64 sequences x 8192 keys, 16 / 32 rows: D = 128 eights 67 / 122 us,
// sixteens 71 / 97; D = 64 47 / 84 and 39 / 65; one sequence, 4 heads x 32768, D = 64:
// 12.3 / 16.9 and 13.7 / 16.5.
int rows_per_group(int64_t heads, int64_t R, int64_t rounds, int D) {
  auto run = [&](int nt) {
    const int64_t slots = int64_t(device_sms()) * ctas_per_sm(D, nt);
    return (heads * ((R + 8 * nt - 1) / (8 * nt)) * rounds + slots - 1) / slots;
  };
  return 20 * run(1) <= (D == 128 ? 26 : D == 64 ? 33 : 29) * run(2) + 10 ? 1 : 2;
}
int plan(Plan &pl, int64_t B, int Hkv, int64_t R, int64_t kv_len, int D, bool lens) {
  const int rounds = rounds_of(static_cast<int>(kv_len));
  const int64_t lim = int64_t(1) << 30;  // rounds and rows of the list are counted in 32 bits
  if (B >= lim || R >= lim || B * Hkv >= lim / R)
    return fail(Q35_ERR_SHAPE, "attn_q4: too many query rows");
  pl.nt = R > 8 ? rows_per_group(B * Hkv, R, rounds, D) : 1;
  const int64_t n_rg = (R + 8 * pl.nt - 1) / (8 * pl.nt);
  if (rounds * B >= lim / (Hkv * n_rg)) return fail(Q35_ERR_SHAPE, "attn_q4: too many key tiles");
  pl.n_rg = static_cast<int>(n_rg);
  const int groups = static_cast<int>(B * Hkv * n_rg), total = groups * rounds;
  const int slots = device_sms() * ctas_per_sm(D, pl.nt);
  const int cut = total < slots ? total : slots, cut_per = (total + cut - 1) / cut;
  const int each = (groups + slots - 1) / slots, whole = each * rounds;
  const int64_t cost = int64_t(whole) * round_cost((groups + each - 1) / each, D);
  const int64_t cut_cost = int64_t(cut_per) * round_cost(cut, D) + join_cost(B * Hkv * R, lens);
  // A warp per group: its tiles one after the other, but four groups begin and end at a
  // time and no warp is without a tile.  A round of it costs 0.85 of one that four warps
  // share and join (396 shapes, 1 to 1000 keys: the choice is 0.7 % above the best of the
  // three on average; 59 sequences x 8 heads x 272 rows, 44 keys, D = 64: whole 84 us,
  // alone 31; 64 x 8 heads x 8 rows, 64 keys, D = 128: 8.0 and 4.3; 64 x 4 x 8, 128 keys:
  // 5.5 and 6.1).
  const int64_t tiles = rounds_of(static_cast<int>(kv_len), 1);
  const int64_t warp_each = (groups + kWarps * int64_t(slots) - 1) / (kWarps * int64_t(slots));
  const int64_t alone_runs = (groups + kWarps * warp_each - 1) / (kWarps * warp_each);
  pl.alone = tiles * groups < lim &&
             17 * tiles * warp_each * round_cost(alone_runs, D) < 20 * (cost < cut_cost ? cost : cut_cost);
  pl.join = !pl.alone && cut_cost < cost;
  pl.scan = pl.join && lens;
  pl.per = pl.join ? cut_per : whole;
  pl.runs = pl.scan ? cut : (total + pl.per - 1) / pl.per;
  if (pl.alone) {
    pl.per = static_cast<int>(warp_each * tiles);
    pl.runs = static_cast<int>(alone_runs);
  }
  return Q35_OK;
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int64_t q35_attn_q4_workspace(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len,
                                         int D) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || Sq <= 0 || D <= 0) return 0;
  if (Sq >= int64_t(1) << 31) return 0;
  if (kv_len < 0 || kv_len >= (int64_t(1) << 31) - 256) return 0;
  int64_t most = 0;  // of the calls with and without kv_lens
  for (int lens = 0; lens < 2; ++lens) {
    Plan pl;
    if (plan(pl, B, Hkv, Hq / Hkv * Sq, kv_len, D, lens != 0) != Q35_OK || !pl.join) continue;
    const int64_t n = partial_rows(pl.runs, pl.nt) * (static_cast<int64_t>(D) + 2) + B + 1;
    if (n > most) most = n;
  }
  return most;
}

extern "C" int q35_attn_q4_fwd(const void *q, const void *k_codes, const void *k_scales,
                               const void *v_codes, const void *v_scales, void *out, int64_t B,
                               int Hq, int Hkv, int64_t Sq, int64_t kv_len, const int32_t *kv_lens,
                               int64_t cap, int D, int group, float scale, int causal,
                               float *workspace, q35_stream_t stream) {
  const int st = q4::check_cache("attn_q4", k_codes, k_scales, v_codes, v_scales, B, Hkv, D, group,
                                 cap);
  if (st) return st;
  if (Sq < 0 || Sq >= int64_t(1) << 31 || kv_len < 0 || Hq <= 0 || Hq % Hkv != 0)
    return fail(Q35_ERR_SHAPE, "attn_q4: Sq %lld, kv_len %lld, Hq %d, Hkv %d", (long long)Sq,
                (long long)kv_len, Hq, Hkv);
  if (kv_len > cap)
    return fail(Q35_ERR_SHAPE, "attn_q4: %lld rows exceed the capacity %lld", (long long)kv_len,
                (long long)cap);
  if (const int bad = q4::check_scale("attn_q4", scale)) return bad;
  if (B == 0 || Sq == 0) return Q35_OK;
  if (!q || !out) return fail(Q35_ERR_INVALID, "attn_q4: null");
  if (!aligned16(q) || !aligned16(out))
    return fail(Q35_ERR_ALIGN, "attn_q4: q, out not 16-byte aligned");
  const int64_t R = Hq / Hkv * Sq;
  Plan pl;
  const int ps = plan(pl, B, Hkv, R, kv_len, D, kv_lens != nullptr);
  if (ps) return ps;
  if (pl.join && !workspace) return fail(Q35_ERR_INVALID, "attn_q4: no workspace");
  if (pl.join && !aligned16(workspace))
    return fail(Q35_ERR_ALIGN, "attn_q4: workspace not 16-byte aligned");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "attn_q4: no device error word");
  Params p{};
  p.q = static_cast<const uint16_t *>(q);
  p.c = Cache{static_cast<uint32_t *>(const_cast<void *>(k_codes)),
              static_cast<uint32_t *>(const_cast<void *>(k_scales)),
              static_cast<uint32_t *>(const_cast<void *>(v_codes)),
              static_cast<uint32_t *>(const_cast<void *>(v_scales))};
  p.out = static_cast<uint16_t *>(out);
  p.ws = workspace;
  p.kv_lens = kv_lens;
  p.err = err;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.Sq = static_cast<int>(Sq);
  p.R = static_cast<int>(R);
  p.n_rg = pl.n_rg;
  p.B = static_cast<int>(B);
  p.runs = pl.runs;
  p.per = pl.per;
  p.scan = pl.scan ? 1 : 0;
  p.causal = causal ? 1 : 0;
  p.kv_len = static_cast<int>(kv_len);
  p.cap = cap;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int64_t rows = B * Hkv * R;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto d, auto gs, auto nt) -> int {
    auto *kern = pl.alone ? &attn_q4_kernel<d(), gs(), nt(), 1> : &attn_q4_kernel<d(), gs(), nt(), kWarps>;
    constexpr int smem = Layout<d(), gs(), nt()>::kSmem;
    const int e = ensure_smem_attr(reinterpret_cast<const void *>(kern), smem);
    if (e) return e;
    Q35_CHECK_CUDA(launch_early(kern, dim3(pl.runs), dim3(kThreads), smem, s, p));
    Q35_LAUNCH_CHECK("attn_q4 launch");
    if (pl.join) {
      // about runs / groups partials a row: 1 or 2, around a dozen, a hundred
      const int64_t each = pl.runs / (B * Hkv * pl.n_rg);
      auto *join = each < 4    ? &attn_q4_join_kernel<d(), 2, 2>
                   : each < 32 ? &attn_q4_join_kernel<d(), 8, 2>
                               : &attn_q4_join_kernel<d(), 16, 8>;
      Q35_CHECK_CUDA(launch_early(join, dim3(static_cast<unsigned>(rows)),
                                  dim3(each < 4 ? 64 : each < 32 ? 256 : 512), 0, s, p, 8 * nt()));
      Q35_LAUNCH_CHECK("attn_q4 join launch");
    }
    return Q35_OK;
  };
  using std::integral_constant;
  auto by_nt = [&](auto d, auto gs) {
    return pl.nt == 2 ? go(d, gs, integral_constant<int, 2>{}) : go(d, gs, integral_constant<int, 1>{});
  };
  integral_constant<int, 128> c128;
  integral_constant<int, 64> c64;
  integral_constant<int, 32> c32;
  if (D == 128) return group == 128 ? by_nt(c128, c128) : group == 64 ? by_nt(c128, c64) : by_nt(c128, c32);
  if (D == 64) return group == 64 ? by_nt(c64, c64) : by_nt(c64, c32);
  return by_nt(c32, c32);
}
