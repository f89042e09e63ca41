// Causal attention of a chunk over an 8-bit paged cache with a scale for each
// (block, head).
//
// Row (j, r) of kv head h (query head h * ratio + r, chunk token j) attends keys
// 0 .. start + j:  z_i = scale * s_k(i) * (q . k_i),  p = softmax(z),
// o = sum_i p_i s_v(i) v_i,  with k_i, v_i the decoded codes and s_k, s_v the
// scales of key i's block. Scores, the running maximum and sum and the output are
// held in fp32.
#include "fp8_heads.h"

using namespace spv;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct HeadAttn {
  void* out;
  const void* q;
  const uint8_t* kpool;
  const uint8_t* vpool;
  const float* scales;
  const int32_t* tables;
  const int32_t* seq_ids;
  const int32_t* start;
  const int32_t* lens;
  int32_t* ctr;
  int maxb, B, C, Hq, Hkv, ratio, d, bs, layer, cap, max_ctx;
  float scale_log2;
};

// A read the contract forbids is recorded as 1 + the entry's index; such a page
// reads block 0 instead.
__device__ __forceinline__ void flag_read(const HeadAttn& p, int b) {
  if (p.ctr) p.ctr[CTR_BAD_READ] = b + 1;
}
__device__ __forceinline__ int block_of(const HeadAttn& p, int sid, int blk, int b) {
  const int id = p.tables[(size_t)sid * p.maxb + min(blk, p.maxb - 1)];
  if ((unsigned)id < (unsigned)p.cap) return id;
  flag_read(p, b);
  return 0;
}

// One wave per row, 64 keys at a time, any head_dim, block size and ratio.
constexpr int kAnyRows = 4;
template <int QT>
__global__ __launch_bounds__(64 * kAnyRows) void head_attn_any_kernel(HeadAttn p, int groups) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ float s_w[kAnyRows][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = p.d;
  const int g = blockIdx.x % groups, bh = blockIdx.x / groups, h = bh % p.Hkv, b = bh / p.Hkv;
  const int row = g * kAnyRows + wave, start = p.start[b], sid = p.seq_ids[b];
  if (g == 0 && h == 0 && threadIdx.x == 0 &&
      (start < 0 || start + p.C > p.max_ctx || (p.lens && start + p.C > p.lens[sid])))
    flag_read(p, b);
  if (row >= p.C * p.ratio) return;  // whole waves; no barrier below
  const int j = row / p.ratio, hq = h * p.ratio + row - j * p.ratio;
  float* const q = reinterpret_cast<float*>(lds) + (size_t)wave * 2 * d;
  float* const o = q + d;
  const size_t at = (((size_t)b * p.C + j) * p.Hq + hq) * d;
  for (int e = lane; e < d; e += 64) {
    q[e] = load_elem<QT>(p.q, at + e) * p.scale_log2;
    o[e] = 0.f;
  }
  const int n = min(start + j + 1, p.max_ctx);
  float m = -INFINITY, l = 0.f;
  for (int base = 0; base < n; base += 64) {
    const int key = base + lane;
    float z = -INFINITY, vs = 0.f;
    if (key < n) {
      const int blk = key / p.bs, off = key - blk * p.bs, phys = block_of(p, sid, blk, b);
      const float* const s = p.scales + scale_of(p.layer, p.cap, phys, p.Hkv, h);
      const uint8_t* const k = p.kpool + page_of(p.layer, p.cap, phys, p.Hkv, h, p.bs, d) + (size_t)off * d;
      float dot = 0.f;
      for (int e = 0; e < d; ++e) dot = fmaf(q[e], fp8e4m3_to_f32(k[e]), dot);
      z = dot * s[0];
      vs = s[1];
    }
    float top = z;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    const float w = exp2f(z - ref), keep = exp2f(m - ref);
    float sum = w;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    l = l * keep + sum;
    m = mn;
    s_w[wave][lane] = w * vs;
    __builtin_amdgcn_wave_barrier();
    for (int e = lane; e < d; e += 64) {
      float acc = o[e] * keep;
      for (int i = 0; i < min(64, n - base); ++i) {
        const int blk = (base + i) / p.bs, off = base + i - blk * p.bs, phys = block_of(p, sid, blk, b);
        const uint8_t* const v = p.vpool + page_of(p.layer, p.cap, phys, p.Hkv, h, p.bs, d);
        acc = fmaf(s_w[wave][i], fp8e4m3_to_f32(v[(size_t)e * p.bs + off]), acc);
      }
      o[e] = acc;
    }
    __builtin_amdgcn_wave_barrier();
  }
  const float inv = n > 0 ? 1.f / l : 0.f;
  for (int e = lane; e < d; e += 64) store_elem<QT>(p.out, at + e, o[e] * inv);
}


// ---------------------------------------------------------------- matrix cores
//
// Head dims 64 and 128, blocks of whole 16-token units. A workgroup of 8 waves
// takes a piece: rows R = 16 RT of one kv head of one entry (all of them, for
// verify chunks) times a range of steps of 64 keys, its waves every eighth step.
// Pages go from HBM to LDS by themselves (loads with an LDS destination), a step
// ahead per wave, and each wave waits for its own; no barrier while it walks.
// Everything stays transposed, so that no value changes lanes between the two
// products:
//   S^T = K Q^T: A = 16 keys x 32 dims, codes converted exactly (every e4m3 value
//     is a bf16 and an fp16 value), B = 16 rows. Lane (g, c) = (lane / 16,
//     lane % 16) gets keys 4 g + i of each of the four tiles for row c. The key that
//     row r of tile t stands for is chosen, token 4 t + r % 4 of unit r / 4 of the
//     step, so that a lane's 16 keys are unit g: one block, one pair of scales.
//   O^T += V^T P^T: A = 16 dims x 32 keys, a lane's keys 8 bytes of a V^T row, B = the
//     lane's own weights.
// K's 16-byte pieces lie in LDS in an order (an exclusive or of a piece's number with
// its row's and unit's) that puts the 16 rows of an operand on different banks.
// The block's K scale multiplies the scores, its V scale the weights. The maximum of
// a row is raised (and O rescaled) only where a step passes it by more than 2^8 (2^3
// for bf16 queries).
// Roundings: scores, sums and O are fp32. A weight meets V in 16 bits:
//   bf16 queries: one part of fp16 (2^-11, an eighth of the output's own rounding),
//     shifted up by 2^11 with V's scale in [1, 2); the scale's power of two goes into
//     V's conversion, against a unit of O's that follows the largest. The second part
//     of bf16 that this saves cost 4 us of 54 at 16 contexts of 32,768 keys. Weights
//     below 2^-25 of the row's largest lose bits, 2^-36 of it each: with values up to
//     2^kNear of the others' no more than an fp32 step of what the largest adds.
//   fp16 queries: two parts of bf16 (2^-17), 8 bits each and of fp32's range.
//   fp32 queries: three parts, and three of each query, in S.
// Steps with masked keys, and all behind the first scales too far apart for that, take
// the parts of bf16, whose range is fp32's (V's scale may be of any size there).

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8, kTileThreads = 64 * kWaves;
constexpr int kGrid = 256;       // one workgroup per CU
constexpr int kStep = 64;        // keys of a step: four units
constexpr int kMinSteps = 8;     // a piece has a step for each wave, where contexts are cut
// What a segment costs beside its steps (look-ups, queries, the join of the waves), in steps, where shares of many
// segments are cut: 128 entries of 32 to 8,192 keys went from 140 to 91 us with it (the slowest workgroup had the
// most segments).
constexpr int kHead = 24;
constexpr float kLowest = -3.402823466e38f;

struct HeadPlan {  // host-chosen shape of a tiled call
  int RT, RG, rpg, D, upb, equal;  // row tiles, row groups, rows of one, head_dim, units per block, pieces of equal length
  int pair;                   // two row groups, walked side by side by workgroups 8 apart
  unsigned upb_magic;         // floor(2^32 / upb) + 1
  int aligned;                // q and out on 16-byte addresses
  int* counters;              // kGrid: arrivals of a segment's parts
  float* part;                // slots of R x D sums and R x (maximum, sum)
};

template <int QT>
struct Parts {
  static constexpr int Q = QT == SPV_F32 ? 3 : 1, P = QT == SPV_F32 ? 3 : 2;
  static constexpr bool half = QT == SPV_BF16;     // weights in one part of fp16
  static constexpr float lift = half ? 3.f : 8.f;  // log2 by which a step may pass the row's maximum
};
constexpr int kHalfShift = 11;  // weights in fp16 are shifted by it: up to 2^3 * 2 * 2^11, bits lost below 2^-25
// V scales of a wave's blocks that fp16 weights meet lie within it (in powers of two). With steps compared to the
// largest scale alone, keys of weight 2^-30.5 and values 2^40 of the others', nearly all of the output, were 2 % off,
// and those of 2^-45.3 and 2^60 lost. Scales 2^14 apart cost the parts of bf16, 61 us for 48 over 16 contexts of 32,768
// keys (D = 64), 102 for 88 at 128 of 32 to 8,192 (D = 128); 2^8 apart they cost nothing.
constexpr int kNear = 12, kUnitLag = 7;  // O's unit is 2^kUnitLag below the largest scale at most
constexpr int kNoScale = -200, kNoUnit = -1000;  // exponents of a scale of 0, of O before the first step

template <bool HI>
__device__ __forceinline__ uint32_t to_bf16x2(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t to_f16x2(uint32_t w, float power) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, HI));
}
// Eight codes as an operand; in fp16 times a power of two from 2^-kNear to 2^kUnitLag, exactly (448 * 2^7 < 65504, and
// every product is a multiple of 2^-21).
template <bool F16>
__device__ __forceinline__ u32x4_t operand(uint32_t a, uint32_t b, float power = 1.f) {
  if constexpr (F16)
    return u32x4_t{to_f16x2<false>(a, power), to_f16x2<true>(a, power), to_f16x2<false>(b, power), to_f16x2<true>(b, power)};
  else return u32x4_t{to_bf16x2<false>(a), to_bf16x2<true>(a), to_bf16x2<false>(b), to_bf16x2<true>(b)};
}
template <bool F16>
__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// The high bit of every byte of w that is a NaN code.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}

// A barrier for what the workgroup keeps in LDS: stores and loads to LDS that are under way stay so.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 16 bytes per lane from memory to LDS: lane l's go to `to` + 16 l; OFF moves both ends.
template <int OFF>
__device__ __forceinline__ void page_to_lds(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, OFF, 0);
}
template <int N>
__device__ __forceinline__ void wait_loads() {  // all but the newest N vector memory operations of the wave
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Four 16-byte pieces from LDS, STEP bytes apart: read in assembly, whose wait is its own, for the compiler would wait
// for every load to LDS before a read of it.
template <int O, int STEP>
__device__ __forceinline__ void lds_read4(u32x4_t (&w)[4], uint32_t a) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%5\n\tds_read_b128 %1, %4 offset:%6\n\t"
      "ds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %4 offset:%8\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
      : "v"(a), "n"(O), "n"(O + STEP), "n"(O + 2 * STEP), "n"(O + 3 * STEP)
      : "memory");
}

// Keys that the rows of group rg of an entry see (a pair's groups are walked as far as the second sees), and steps of
// them (one at least).
__device__ __forceinline__ int group_keys(const HeadAttn& p, const HeadPlan& pl, int start, int rg) {
  const int last = pl.pair || rg == pl.RG - 1 ? p.C - 1 : min(p.C - 1, (rg * pl.rpg + pl.rpg - 1) / p.ratio);
  return min(start + last + 1, p.max_ctx);
}
__device__ __forceinline__ int group_steps(const HeadAttn& p, const HeadPlan& pl, int start, int rg) {
  return max(1, (group_keys(p, pl, start, rg) + kStep - 1) / kStep);
}

template <int QT, int D, int RT>
__global__ __launch_bounds__(kTileThreads, 2) void head_attn_tile_kernel(HeadAttn p, HeadPlan pl) {
  constexpr bool F16 = QT == SPV_F16, kF16W = Parts<QT>::half;
  constexpr int NQ = Parts<QT>::Q, NP = Parts<QT>::P, R = RT * 16, NCH = D / 32, NDT = D / 16;
  constexpr int kUnit = 16 * D, kHalf = 4 * kUnit;  // bytes of a unit, of a step's K or V
  constexpr int NK = kHalf / 1024;                                           // loads of a step's K, or V
  // The waves' sums are joined in as many dims at once as fit where the pages were (at least 64).
  constexpr int kColPad = 4, kCols = D == 64 || R * (D + kColPad) * 4 <= 2 * kHalf ? D : 64;
  constexpr int kStage = 2 * kHalf > R * (kCols + kColPad) * 4 ? 2 * kHalf : R * (kCols + kColPad) * 4;
  constexpr bool kQReg = RT * NCH * NQ <= 4;  // queries in registers, where they are few
  __shared__ __align__(1024) uint8_t s_page[kWaves * kStage];  // [wave][K | V]; the waves' sums later
  __shared__ __align__(16) u32x4_t s_q[NQ * RT * NCH * 64];
  __shared__ float s_ml[2][kWaves][R];
  __shared__ float s_row[2][R];  // joined maximum and sum
  __shared__ int s_nan[D];       // first key whose value is NaN in a dim, where rows end
  __shared__ int s_last;
  // A pair's workgroups are on one XCD (its L2 has the pages for the second): half 0 and 1 of a worker.
  const int worker = pl.pair ? (int)(blockIdx.x >> 4) * 8 + (int)(blockIdx.x & 7) : (int)blockIdx.x;
  const int half = pl.pair ? (int)(blockIdx.x >> 3) & 1 : 0, workers = pl.pair ? kGrid / 2 : kGrid;
  const int counted = pl.pair ? 1 : pl.RG;  // row groups that count for themselves
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;

  // ---- which piece: the waves work it out alike, each lane for epl entries (the first two kept). Steps of an entry,
  // or pieces of at most P steps; equal = 0: shares of all steps in a row.
  const int epl = (p.B + 63) >> 6, b0 = min(lane * epl, p.B), b1 = min(b0 + epl, p.B);
  int st[2], id[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = min(b0 + i, p.B - 1);
    st[i] = p.start[b];
    id[i] = p.seq_ids[b];
  }
  const int head = pl.equal ? 0 : kHead;
  // Pieces that n steps go into, at about 1 / inv steps each.
  auto pieces = [](int n, float inv) { return max(1, (int)ceilf((float)n * inv)); };
  float inv_p = 0.f;
  auto count = [&](int start) {
    int n = 0;
    for (int rg = 0; rg < counted; ++rg) {
      const int k = group_steps(p, pl, start, rg);
      n += pl.equal ? pieces(k, inv_p) : k + head;
    }
    return n * p.Hkv;
  };
  int P = kMinSteps;
  if (pl.equal) {  // two entries a lane at most: there are no more segments than half the workers
    int steps = 0;
    for (int rg = 0; rg < counted; ++rg) {
      if (b0 < b1) steps += group_steps(p, pl, st[0], rg);
      if (b0 + 1 < b1) steps += group_steps(p, pl, st[1], rg);
    }
    P = max((lane63(wave_incl_sum(steps)) * p.Hkv + workers - 1) / workers, kMinSteps);
    // The smallest P that leaves no more pieces than workers, eight candidates at a time; ends at the latest with one
    // piece per segment.
    constexpr int kTry = 8;
    for (bool found = false; !found;) {
      float inv[kTry];
      int n[kTry], sizes[kTry];
#pragma unroll
      for (int i = 0; i < kTry; ++i) {
        sizes[i] = P + max(1, P >> 4) * i;
        inv[i] = __builtin_amdgcn_rcpf((float)sizes[i]);
        n[i] = 0;
      }
      for (int rg = 0; rg < counted; ++rg) {
        const int k0 = b0 < b1 ? group_steps(p, pl, st[0], rg) : 0, k1 = b0 + 1 < b1 ? group_steps(p, pl, st[1], rg) : 0;
#pragma unroll
        for (int i = 0; i < kTry; ++i) n[i] += (k0 ? pieces(k0, inv[i]) : 0) + (k1 ? pieces(k1, inv[i]) : 0);
      }
#pragma unroll
      for (int i = 0; i < kTry; ++i) n[i] = lane63(wave_incl_sum(n[i])) * p.Hkv;
#pragma unroll
      for (int i = kTry - 1; i >= 0; --i)
        if (n[i] <= workers) {
          found = true;
          inv_p = inv[i];
        }
      P = sizes[kTry - 1] + 1;
    }
  }
  const int v0 = b0 < b1 ? count(st[0]) : 0;  // of the lane's first entry; of all its entries
  int mine = v0 + (b0 + 1 < b1 ? count(st[1]) : 0);
  for (int b = b0 + 2; b < b1; ++b) mine += count(p.start[b]);
  const int upto = wave_incl_sum(mine), total = lane63(upto);
  if (!pl.equal) P = max((total + workers - 1) / workers, kMinSteps);
  const int x0 = pl.equal ? worker : worker * P;
  const int x1 = min(total, pl.equal ? x0 + 1 : x0 + P);
  if (blockIdx.x == kGrid - 1 && wave == 0) {
    for (int b = b0; b < b1; ++b) {
      const int start = p.start[b];
      if (start < 0 || start + p.C > p.max_ctx || (p.lens && start + p.C > p.lens[p.seq_ids[b]])) flag_read(p, b);
    }
  }

  for (int cur = x0; cur < x1;) {
    lds_barrier();
    const int owner = __ffsll((unsigned long long)__ballot(upto > cur)) - 1;
    int off = cur - __builtin_amdgcn_readlane(upto - mine, owner), b = owner * epl, start, sid;
    if (epl <= 2) {
      const int first = __builtin_amdgcn_readlane(v0, owner);
      const bool second = off >= first;
      if (second) off -= first;
      b += second;
      start = __builtin_amdgcn_readlane(second ? st[1] : st[0], owner);
      sid = __builtin_amdgcn_readlane(second ? id[1] : id[0], owner);
    } else {  // the owner's entries, 64 at a time
      for (int e0 = 0;; e0 += 64) {
        const bool in = e0 + lane < epl && b + lane < p.B;
        const int s1 = p.start[min(b + lane, p.B - 1)], n = in ? count(s1) : 0;
        const int sum = wave_incl_sum(n);
        if (off < lane63(sum)) {
          const int at = __ffsll((unsigned long long)__ballot(sum > off)) - 1;
          off -= __builtin_amdgcn_readlane(sum - n, at);
          b += at;
          start = __builtin_amdgcn_readlane(s1, at);
          break;
        }
        off -= lane63(sum);
        b += 64;
      }
      sid = p.seq_ids[b];
    }
    int rg = 0, n = 0, k = 0;
    for (;; ++rg) {
      n = group_steps(p, pl, start, rg);
      k = pl.equal ? pieces(n, inv_p) : n + head;
      if (off < k * p.Hkv || rg == counted - 1) break;
      off -= k * p.Hkv;
    }
    const int h = off / k, i_in = off - h * k;
    int first, last, nparts, my, slot0;  // steps [first, last); parts of the segment, which is this; slots
    if (pl.equal) {
      const int each = n / k, more = n - each * k;
      first = i_in * each + min(i_in, more);
      last = first + each + (i_in < more);
      nparts = k;
      my = i_in;
      slot0 = cur - i_in;
      cur = x1;
    } else {
      first = max(0, i_in - head);
      const int take = min(k - i_in, x1 - cur);
      last = i_in + take - head;
      slot0 = cur - i_in + head;  // the segment's first step among all
      nparts = (slot0 + n - 1) / P - slot0 / P + 1;
      my = worker - slot0 / P;
      cur += take;
      if (last <= first) continue;  // the share ends before the segment's first step
    }
    if (pl.pair) rg = half;
    // Slot of part i: its worker's first or second one (a share's first piece, or its last).
    auto slot_of = [&](int i) {
      const int w = pl.equal ? slot0 + i : slot0 / P + i;
      return 2 * (half * workers + w) + (!pl.equal && w * P < slot0);
    };
    const int keys = group_keys(p, pl, start, rg), units = max(1, (keys + 15) >> 4);
    const int row0 = rg * pl.rpg, rows = min(pl.rpg, p.C * p.ratio - row0);
    const int32_t* const table = p.tables + (size_t)sid * p.maxb;
    const size_t page_bytes = (size_t)p.bs * D, block_bytes = page_bytes * p.Hkv;
    const uint8_t* const kbase = p.kpool + ((size_t)p.layer * p.cap * p.Hkv + h) * page_bytes;
    const uint8_t* const vbase = p.vpool + ((size_t)p.layer * p.cap * p.Hkv + h) * page_bytes;
    const float* const sbase = p.scales + ((size_t)p.layer * p.Hkv + h) * p.cap * 2;

    // ---- the wave's pages. Lane i holds what unit i % 4 of step i / 4 of its next 16 steps needs: where it lies and
    // its scales.
    const int steps = last - first > wave ? (last - first - wave + kWaves - 1) / kWaves : 0;  // of this wave
    auto step_at = [&](int k) { return first + wave + k * kWaves; };
    uint32_t l_k[2] = {0, 0}, l_v[2] = {0, 0};  // byte offsets of the unit's K and V, in halves
    float2 l_scale = {0.f, 0.f};
    auto look_up = [&](int k) {  // for steps k .. k + 15
      const int u = min(step_at(k + (lane >> 2)) * 4 + (lane & 3), units - 1);
      const int blk = pl.upb == 1 ? u : (int)__umulhi((unsigned)u, pl.upb_magic);
      const int tok = (u - blk * pl.upb) * 16;
      int block = table[min(blk, p.maxb - 1)];
      if ((unsigned)block >= (unsigned)p.cap) {
        if (lane >> 2 < steps - k) flag_read(p, b);
        block = 0;
      }
      l_scale = *reinterpret_cast<const float2*>(sbase + (size_t)block * 2);
      const size_t at = (size_t)block * block_bytes, ka = at + (size_t)tok * D, va = at + tok;
      l_k[0] = (uint32_t)ka;
      l_k[1] = (uint32_t)(ka >> 32);
      l_v[0] = (uint32_t)va;
      l_v[1] = (uint32_t)(va >> 32);
    };
    // The unit's address, in scalar registers.
    auto unit_from = [&](const uint8_t* base, const uint32_t (&l)[2], int at) {
      uint64_t a = (uint64_t)base + ((uint64_t)__builtin_amdgcn_readlane(l[1], at) << 32 | (uint32_t)__builtin_amdgcn_readlane(l[0], at));
      asm("" : "+s"(a));
      return reinterpret_cast<const uint8_t*>(a);
    };
    uint8_t* const stage0 = s_page + wave * kStage;
    // Lane offsets of a K load (row, piece: exclusive or with 32 u for unit u) and of a V load (row).
    const int krow = D == 128 ? lane >> 3 : lane >> 2;
    const uint32_t kvoff = D == 128 ? krow * 128 + (((lane & 7) ^ ((krow >> 1) & 1)) * 16) : krow * 64 + (lane & 3) * 16;
    const uint32_t vvoff = (uint32_t)lane * (uint32_t)p.bs;
    float2 sc = {0.f, 0.f};  // scales of the lane's keys of the step ahead
    auto fetch_k = [&](int k) {
      if ((k & 15) == 0) look_up(k);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = (k & 15) * 4 + u;
        const uint8_t* const from = unit_from(kbase, l_k, at);
        const uint32_t lo = kvoff ^ (D == 128 ? u * 32 : u * 16);
        page_to_lds<0>(from + lo, stage0 + u * kUnit);
        if constexpr (D == 128) page_to_lds<1024>(from + lo, stage0 + u * kUnit);
      }
      const int at = (k & 15) * 4 + g;
      sc = make_float2(__shfl(l_scale.x, at, 64), __shfl(l_scale.y, at, 64));
    };
    auto fetch_v = [&](int k) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = (k & 15) * 4 + u;
        const uint8_t* const from = unit_from(vbase, l_v, at);
        page_to_lds<0>(from + vvoff, stage0 + kHalf + u * kUnit);
        if constexpr (D == 128) page_to_lds<0>(from + (size_t)64 * p.bs + vvoff, stage0 + kHalf + u * kUnit + 1024);
      }
    };
    if (steps > 0) {
      fetch_k(0);
      fetch_v(0);
    }

    // ---- queries to LDS as operands: [part][row tile][chunk][lane] 16 bytes; dims of a chunk as K's pieces go
    if ((int)threadIdx.x < D) s_nan[threadIdx.x] = 0x7fffffff;
    for (int i = threadIdx.x; i < R * (D / 8); i += kTileThreads) {
      const int row = i / (D / 8), piece = i - row * (D / 8), r = row0 + row;
      float x[8];
      if (row < rows) {
        const int j = r / p.ratio, hq = h * p.ratio + r - j * p.ratio;
        const size_t at = (((size_t)b * p.C + j) * p.Hq + hq) * D + piece * 8;
        if (pl.aligned) {
          constexpr int E = Piece<QT>::E;
#pragma unroll
          for (int q = 0; q < 8 / E; ++q) {
            Piece<QT> w;
            w.unpack(reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(p.q) + at * (16 / E))[q]);
#pragma unroll
            for (int e = 0; e < E; ++e) x[q * E + e] = w.x[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = load_elem<QT>(p.q, at + e);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
      }
      if (p.scale_log2 < 0.f) {  // the scores' factor is taken as positive below
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = -x[e];
      }
      const int ch = 2 * (piece >> 3) + (piece & 1), ln = ((piece >> 1) & 3) * 16 + (row & 15);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (F16) {
            w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x[2 * e], x[2 * e + 1]}, f16x2_t));
          } else {
            w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
            x[2 * e] -= __uint_as_float(w[e] << 16);
            x[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
          }
        }
        s_q[((q * RT + (row >> 4)) * NCH + ch) * 64 + ln] = w;
      }
    }
    lds_barrier();
    auto query = [&](int rt, int ch, int q) { return s_q[((q * RT + rt) * NCH + ch) * 64 + lane]; };
    u32x4_t qreg[kQReg ? RT : 1][kQReg ? NCH : 1][kQReg ? NQ : 1];
    if constexpr (kQReg) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
          for (int q = 0; q < NQ; ++q) qreg[rt][ch][q] = query(rt, ch, q);
    }

    f32x4_t o[RT][NDT];
    float m[RT], l[RT];
    int unit_exp = kNoUnit;  // kF16W: O stands for O 2^(unit_exp - kHalfShift)
    int high_exp = kNoUnit, low_exp = -kNoUnit;  // kF16W: of the V scales so far
    int apart = 0;                               // kF16W: they are further apart than kNear, or one is 0
    int seen[RT];  // keys that the lane's row attends
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kLowest;
      l[rt] = 0.f;
      seen[rt] = min(start + min((row0 + rt * 16 + c) / p.ratio, p.C - 1) + 1, p.max_ctx);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[rt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const int all_see = min(start + row0 / p.ratio + 1, p.max_ctx);  // keys that every row attends
    const float factor = fabsf(p.scale_log2);
    // LDS addresses of the lane's operand bytes: K row c % 4 of unit c / 4, piece g; V row c of unit g.
    const uint32_t base0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)stage0;
    const uint32_t kat = base0 + (c >> 2) * kUnit + (c & 3) * D +
                         ((g ^ (D == 128 ? ((c >> 1) & 1) | (c >> 2) << 1 : c >> 2)) * 16);
    const uint32_t vat = base0 + kHalf + g * kUnit + c * 16;

    auto run_step = [&](int k, auto more) {  // more: step k + 1 exists
      const int step = step_at(k);
      const bool masked = (step + 1) * kStep > all_see;
      const float ksc = sc.x * factor, vsc = sc.y;
      const int base = step * kStep + g * 16;  // the lane's first key
      // Weights where no key is masked and the scales allow it: 2^(z - m) and V's scale in one power, for bf16
      // queries what the scale is over a power of two, which goes into V's conversion; their sum is theirs without it.
      // Elsewhere, and for fp32 queries, one after the other and in parts of bf16.
      const int vexp = vsc > 0.f ? __builtin_amdgcn_frexp_expf(vsc) - 1 : kNoScale;  // s_v in [2^vexp, 2^(vexp + 1))
      bool careful = QT == SPV_F32 || masked;
      if constexpr (kF16W) {
        if (__any(vexp > high_exp || vexp < low_exp)) {  // beyond those so far: a few steps of a walk
#pragma unroll
          for (int x = 0; x < 64; x += 16) {
            const int e = __builtin_amdgcn_readlane(vexp, x);
            high_exp = max(high_exp, e);
            low_exp = min(low_exp, e);
          }
          apart = high_exp - low_exp > kNear || low_exp == kNoScale;
          if (high_exp > unit_exp + kUnitLag) {  // O's unit 2^unit_exp follows the scales
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[rt][dt][i] = ldexpf(o[rt][dt][i], unit_exp - high_exp);
            unit_exp = high_exp;
          }
        }
        // Read so that the loop is not made twice, once for each value: 7 registers would be spilled (D = 128).
        careful |= __builtin_amdgcn_readfirstlane(apart) != 0;
      } else {
        careful |= (bool)__any(!(vsc > 0x1p-60f && vsc < 0x1p60f));
      }
      auto body = [&](auto plain, auto more_tag) {
        constexpr bool MORE = decltype(more_tag)::value;
        // s_v times 2^vshift is what a weight takes; in fp16 the part of it in [1, 2), times 2^kHalfShift.
        const float vpart = kF16W ? ldexpf(vsc, kHalfShift - vexp) : vsc;
        const float vlog = __builtin_amdgcn_logf(vpart), vinv = __builtin_amdgcn_rcpf(vpart);
        const float vall = kF16W ? ldexpf(vsc, kHalfShift - unit_exp) : vsc;
        const float vpow = __uint_as_float((uint32_t)(min(max(vexp - unit_exp, -kNear), kUnitLag) + 127) << 23);
        auto lift = [&](int rt, float top) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float mn = fmaxf(m[rt], top), keep = __builtin_amdgcn_exp2f(m[rt] - mn);
          m[rt] = mn;
          l[rt] *= keep;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[rt][dt] *= keep;
        };
        wait_loads<NK>();  // K of this step is there: behind it came its V
        f32x4_t s[RT][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int t = 0; t < 4; ++t) s[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int cc = 0; cc < D / 64; ++cc) {
          u32x4_t kw[4];
          lds_read4<0, 4 * D>(kw, kat ^ (cc * 64));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int ch = 2 * cc + half;
            u32x4_t qv[RT][NQ];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int q = 0; q < NQ; ++q) {
                if constexpr (kQReg) qv[rt][q] = qreg[rt][ch][q];
                else qv[rt][q] = query(rt, ch, q);
              }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const u32x4_t kop = operand<F16>(kw[t][2 * half], kw[t][2 * half + 1]);
#pragma unroll
              for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][t] = mfma<F16>(kop, qv[rt][q], s[rt][t]);
            }
            if constexpr (RT > 2) __builtin_amdgcn_sched_barrier(0);
          }
        }
        if constexpr (MORE) fetch_k(k + 1);
        uint32_t pw[RT][2][NP][4];
        float top[RT];
        if (plain) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            top[rt] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float z = base + i < seen[rt] ? s[rt][i >> 2][i & 3] * ksc : -INFINITY;
              s[rt][i >> 2][i & 3] = z;
              top[rt] = fmaxf(top[rt], z);
            }
          }
        } else {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            top[rt] = s[rt][0][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top[rt] = fmaxf(top[rt], s[rt][i >> 2][i & 3]);
            top[rt] *= ksc;
          }
        }
        bool higher = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) higher |= top[rt] > m[rt] + Parts<QT>::lift;
        if (__any(higher)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) lift(rt, top[rt]);
        }
        if (plain) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float e = __builtin_amdgcn_exp2f(s[rt][i >> 2][i & 3] - m[rt]);
              l[rt] += e;
              s[rt][i >> 2][i & 3] = e * vall;
            }
        } else {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const float off = vlog - m[rt];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float w = __builtin_amdgcn_exp2f(fmaf(s[rt][i >> 2][i & 3], ksc, off));
              s[rt][i >> 2][i & 3] = w;
              sum += w;
            }
            l[rt] = fmaf(sum, vinv, l[rt]);
          }
        }
        if (kF16W && !plain) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              pw[rt][i >> 2][0][i & 3] = pack_f16(s[rt][i >> 1][2 * (i & 1)], s[rt][i >> 1][2 * (i & 1) + 1]);
        } else {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int q = 0; q < NP; ++q)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float x = s[rt][i >> 1][2 * (i & 1)], y = s[rt][i >> 1][2 * (i & 1) + 1];
                const uint32_t u = pack_bf16(x, y);
                pw[rt][i >> 2][q][i & 3] = u;
                if (q + 1 < NP) {
                  s[rt][i >> 1][2 * (i & 1)] = x - __uint_as_float(u << 16);
                  s[rt][i >> 1][2 * (i & 1) + 1] = y - __uint_as_float(u & 0xffff0000u);
                }
              }
        }
        // V of this step is there: behind it came K of the next.
        if constexpr (MORE) wait_loads<NK>();
        else wait_loads<0>();
#pragma unroll
        for (int d4 = 0; d4 < NDT / 4; ++d4) {
          u32x4_t vw[4];
          if (d4 == 0) lds_read4<0, 256>(vw, vat);
          else lds_read4<1024, 256>(vw, vat);
          if (masked) {  // values behind the rows' last key are not looked at
            const int valid = keys - base;
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int nb = min(max(valid - 4 * i, 0), 4);
              const uint32_t in = nb == 4 ? 0xffffffffu : (1u << (8 * nb)) - 1u;
#pragma unroll
              for (int dt = 0; dt < 4; ++dt) {
                vw[dt][i] &= in;
                bad |= nan_codes(vw[dt][i]);
              }
            }
            // A NaN among the chunk's own values reaches the rows that see it, and no other: it is taken out here, and
            // what remembers it is the first key of each dim that holds one.
            if (__any(bad != 0)) {
#pragma unroll
              for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t w = nan_codes(vw[dt][i]);
                  if (w) atomicMin(&s_nan[(4 * d4 + dt) * 16 + c], base + 4 * i + (__ffs(w) >> 3) - 1);
                  vw[dt][i] &= ~((w >> 7) * 0xffu);
                }
            }
          }
#pragma unroll
          for (int mm = 0; mm < 2; ++mm) {  // eight sums in turn, so that none waits for its last addition
            auto weights = [&](int rt, int q) {
              return u32x4_t{pw[rt][mm][q][0], pw[rt][mm][q][1], pw[rt][mm][q][2], pw[rt][mm][q][3]};
            };
            u32x4_t vop[4];
            if (kF16W && !plain) {
#pragma unroll
              for (int dt = 0; dt < 4; ++dt) vop[dt] = operand<true>(vw[dt][2 * mm], vw[dt][2 * mm + 1], vpow);
#pragma unroll
              for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][4 * d4 + dt] = mfma<true>(vop[dt], weights(rt, 0), o[rt][4 * d4 + dt]);
            } else {
#pragma unroll
              for (int dt = 0; dt < 4; ++dt) vop[dt] = operand<false>(vw[dt][2 * mm], vw[dt][2 * mm + 1]);
#pragma unroll
              for (int q = NP - 1; q >= 0; --q)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                  for (int rt = 0; rt < RT; ++rt) o[rt][4 * d4 + dt] = mfma<false>(vop[dt], weights(rt, q), o[rt][4 * d4 + dt]);
            }
          }
        }
        if constexpr (MORE) fetch_v(k + 1);
      };
      // A body of its own for the ordinary steps (16 contexts of 32,768 keys, D = 64: 46.5 us, 49.3 without), where
      // registers allow two: at D = 128 they spill (91 us become 132 at 128 contexts of 32 to 8,192 keys).
      if constexpr (QT == SPV_F32) body(std::true_type{}, more);
      else if constexpr (D > 64) body(careful, more);
      else if (careful) body(std::true_type{}, more);
      else body(std::false_type{}, more);
    };
    int k_step = 0;
    for (; k_step + 1 < steps; ++k_step) run_step(k_step, std::true_type{});
    for (; k_step < steps; ++k_step) run_step(k_step, std::false_type{});

    // ---- the waves' sums, joined in their order
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += __shfl_xor(l[rt], 16, 64);
      l[rt] += __shfl_xor(l[rt], 32, 64);
      if (g == 0) {
        s_ml[0][wave][rt * 16 + c] = m[rt];
        s_ml[1][wave][rt * 16 + c] = l[rt];
      }
    }
    lds_barrier();
    float keep[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = kLowest;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, s_ml[0][w][rt * 16 + c]);
      keep[rt] = __builtin_amdgcn_exp2f(m[rt] - mx);
      if constexpr (kF16W) keep[rt] = ldexpf(keep[rt], unit_exp - kHalfShift);
      if (wave == 0 && g == 0) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          sum = fmaf(s_ml[1][w][rt * 16 + c], __builtin_amdgcn_exp2f(s_ml[0][w][rt * 16 + c] - mx), sum);
        s_row[0][rt * 16 + c] = mx;
        s_row[1][rt * 16 + c] = sum;
      }
    }
    const bool whole = nparts == 1;
    constexpr size_t kSlot = (size_t)R * (D + 2);  // floats of a slot
    const __amdgpu_buffer_rsrc_t slot_rsrc = coherent_rsrc(pl.part + (whole ? 0 : (size_t)slot_of(my) * kSlot));
    // Four dims of a row, normalised, to the output.
    auto put = [&](int row, int e, f32x4_t v, float sum) {
      const int r = row0 + row, j = r / p.ratio, hq = h * p.ratio + r - j * p.ratio;
      const float inv = min(start + j + 1, p.max_ctx) > 0 ? 1.f / sum : 0.f;
      const size_t at = (((size_t)b * p.C + j) * p.Hq + hq) * D + e;
      if (!pl.aligned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store_elem<QT>(p.out, at + i, v[i] * inv);
      } else if constexpr (QT == SPV_F32) {
        *reinterpret_cast<f32x4_t*>(static_cast<float*>(p.out) + at) = v * inv;
      } else {
        u32x2_t w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (F16) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * i] * inv, v[2 * i + 1] * inv}, f16x2_t));
          else w[i] = pack_bf16(v[2 * i] * inv, v[2 * i + 1] * inv);
        }
        asm("" : "+v"(w));
        *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + at) = w;
      }
    };
    float* const s_o = reinterpret_cast<float*>(s_page);  // [wave][row][kCols + pad]
#pragma unroll
    for (int pass = 0; pass < D / kCols; ++pass) {
      if (pass) lds_barrier();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < kCols / 16; ++dt)
          *reinterpret_cast<f32x4_t*>(s_o + (wave * R + rt * 16 + c) * (kCols + kColPad) + dt * 16 + 4 * g) =
              o[rt][pass * (kCols / 16) + dt] * keep[rt];
      lds_barrier();
      for (int i = threadIdx.x; i < rows * (kCols / 4); i += kTileThreads) {
        const int row = i / (kCols / 4), e = (i - row * (kCols / 4)) * 4;
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          sum += *reinterpret_cast<const f32x4_t*>(s_o + (w * R + row) * (kCols + kColPad) + e);
        const int sees = min(start + (row0 + row) / p.ratio + 1, p.max_ctx);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (s_nan[pass * kCols + e + j] < sees) sum[j] = __uint_as_float(0x7fc00000u);
        if (whole) put(row, pass * kCols + e, sum, s_row[1][row]);
        else store_coherent_b128(slot_rsrc, ((size_t)row * D + pass * kCols + e) * 4, __builtin_bit_cast(u32x4_t, sum));
      }
    }
    if (whole) continue;
    if ((int)threadIdx.x < R)
      store_coherent_b64(slot_rsrc, ((size_t)R * D + threadIdx.x * 2) * 4,
                         u32x2_t{__float_as_uint(s_row[0][threadIdx.x]), __float_as_uint(s_row[1][threadIdx.x])});
    // Counted at the workgroup in which the segment begins: it begins one segment at most that others go on with.
    if (!arrive_last(pl.counters + half * workers + (pl.equal ? slot0 : slot0 / P), nparts, &s_last)) continue;

    // ---- the segment's last workgroup joins its parts, in their order: kAt parts of all the thread's pieces in flight
    constexpr int kItems = (R * (D / 4) + kTileThreads - 1) / kTileThreads, kAt = 4;
    f32x4_t acc[kItems];
    float mx[kItems], sums[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      mx[i] = kLowest;
      sums[i] = 0.f;
    }
    for (int q0 = 0; q0 < nparts; q0 += kAt) {
      u32x4_t v[kAt][kItems];
      u32x2_t ml[kAt][kItems];
#pragma unroll
      for (int q = 0; q < kAt; ++q) {
        const __amdgpu_buffer_rsrc_t r = coherent_rsrc(pl.part + (size_t)slot_of(min(q0 + q, nparts - 1)) * kSlot);
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const int row = min((int)threadIdx.x + i * kTileThreads, R * (D / 4) - 1) / (D / 4);
          v[q][i] = load_coherent_b128(r, (size_t)min((int)threadIdx.x + i * kTileThreads, R * (D / 4) - 1) * 16);
          ml[q][i] = load_coherent_b64(r, ((size_t)R * D + row * 2) * 4);
        }
      }
#pragma unroll
      for (int q = 0; q < kAt; ++q) {
        if (q0 + q >= nparts) break;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const float mq = __uint_as_float(ml[q][i][0]), mn = fmaxf(mx[i], mq);
          const float was = __builtin_amdgcn_exp2f(mx[i] - mn), is = __builtin_amdgcn_exp2f(mq - mn);
          mx[i] = mn;
          sums[i] = fmaf(__uint_as_float(ml[q][i][1]), is, sums[i] * was);
          acc[i] = acc[i] * was + __builtin_bit_cast(f32x4_t, v[q][i]) * is;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int at = threadIdx.x + i * kTileThreads, row = at / (D / 4);
      if (row < rows) put(row, (at - row * (D / 4)) * 4, acc[i], sums[i]);
    }
  }
}

// Which shape a call takes, or false: the kernel of one wave per row.
bool tile_plan(int32_t B, int32_t C, int32_t Hq, int32_t Hkv, int32_t d, int32_t bs, int32_t max_ctx, HeadPlan& pl) {
  if ((d != 64 && d != 128) || bs % 16 || B < 1) return false;
  const int ratio = Hq / Hkv;
  const long long rows = (long long)C * ratio;
  if (rows > 0x3fffffffLL) return false;
  pl.D = d;
  pl.RG = (int)((rows + 31) / 32);
  pl.rpg = (int)((rows + pl.RG - 1) / pl.RG);
  pl.RT = (pl.rpg + 15) / 16;
  pl.pair = pl.RG == 2;
  pl.upb = bs / 16;
  pl.upb_magic = (unsigned)(0x100000000ULL / (unsigned)pl.upb + 1);
  const long long segs = (long long)B * (pl.pair ? 1 : pl.RG) * Hkv, steps = ((long long)max_ctx + kStep - 1) / kStep + kHead;
  if (segs * steps > 0x3fffffffLL || ((long long)max_ctx / 16 + 1) * pl.upb > 0x7fffffffLL) return false;
  pl.equal = segs * 2 <= (pl.pair ? kGrid / 2 : kGrid);
  return true;
}

constexpr size_t kCounterBytes = SPV_HEADS_COUNTER_BYTES;  // at the same place for calls of every shape
static_assert(kCounterBytes == kGrid * sizeof(int));
size_t tile_bytes(const HeadPlan& pl) {
  return kCounterBytes + (size_t)2 * kGrid * pl.RT * 16 * (pl.D + 2) * sizeof(float);
}

template <int QT, int D>
void launch_tile(const HeadAttn& p, const HeadPlan& pl, hipStream_t s) {
#define SPV_T(RT) hipLaunchKernelGGL((head_attn_tile_kernel<QT, D, RT>), dim3(kGrid), dim3(kTileThreads), 0, s, p, pl)
  if (pl.RT == 1) SPV_T(1);
  else SPV_T(2);
#undef SPV_T
}

}  // namespace

extern "C" {

size_t spv_verify_attn_fp8_heads_workspace_bytes(int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads,
                                                 int32_t head_dim, int32_t block_size, int32_t max_ctx) {
  HeadPlan pl{};
  if (B < 1 || C < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads || block_size < 1 ||
      max_ctx < 1 || !tile_plan(B, C, num_q_heads, num_kv_heads, head_dim, block_size, max_ctx, pl))
    return 0;
  return tile_bytes(pl);
}

int spv_verify_attn_fp8_heads(void* out, const void* q, int q_dtype, const void* k_pool, const void* v_pool,
                              const float* kv_scales, const int32_t* block_tables, int32_t max_blocks_per_seq,
                              const int32_t* seq_ids, const int32_t* start_pos, const int32_t* seq_lens, int32_t* ctr,
                              int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                              int32_t block_size, int32_t layer, int32_t capacity, int32_t max_ctx, float scale,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (!out || !q || !k_pool || !v_pool || !kv_scales || !block_tables || !seq_ids || !start_pos || B < 0 || C < 1 ||
      num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads || head_dim < 1 || block_size < 1 ||
      layer < 0 || capacity < 1 || max_blocks_per_seq < 1 || max_ctx < 1)
    return SPV_ERR_ARG;
  if (q_dtype != SPV_F32 && q_dtype != SPV_BF16 && q_dtype != SPV_F16) return SPV_ERR_ARG;
  if ((max_ctx + (long long)block_size - 1) / block_size > max_blocks_per_seq) return SPV_ERR_ARG;
  if (head_dim > 2048) return SPV_ERR_UNSUPPORTED;
  const int ratio = num_q_heads / num_kv_heads;
  const long long groups = ((long long)C * ratio + kAnyRows - 1) / kAnyRows, grid = groups * num_kv_heads * B;
  if ((long long)C * ratio > 0x3fffffffLL || grid > 0x7fffffffLL) return SPV_ERR_ARG;
  if (B == 0) return SPV_OK;
  const HeadAttn p{out, q, static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), kv_scales,
                   block_tables, seq_ids, start_pos, seq_lens, ctr, max_blocks_per_seq, B, C, num_q_heads,
                   num_kv_heads, ratio, head_dim, block_size, layer, capacity, max_ctx, scale * kLog2e};
  HeadPlan pl{};
  const bool pools_aligned = ((uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0 && (uintptr_t)kv_scales % 8 == 0;
  if (pools_aligned && tile_plan(B, C, num_q_heads, num_kv_heads, head_dim, block_size, max_ctx, pl)) {
    if (!workspace || workspace_bytes < tile_bytes(pl) || (uintptr_t)workspace % 16) return SPV_ERR_WORKSPACE;
    pl.counters = static_cast<int*>(workspace);
    pl.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
    pl.aligned = ((uintptr_t)q | (uintptr_t)out) % 16 == 0;
    hipStream_t s = (hipStream_t)stream;
    if (head_dim == 64) {
      if (q_dtype == SPV_F32) launch_tile<SPV_F32, 64>(p, pl, s);
      else if (q_dtype == SPV_BF16) launch_tile<SPV_BF16, 64>(p, pl, s);
      else launch_tile<SPV_F16, 64>(p, pl, s);
    } else {
      if (q_dtype == SPV_F32) launch_tile<SPV_F32, 128>(p, pl, s);
      else if (q_dtype == SPV_BF16) launch_tile<SPV_BF16, 128>(p, pl, s);
      else launch_tile<SPV_F16, 128>(p, pl, s);
    }
    SPV_CHECK_LAUNCH();
    return SPV_OK;
  }
  const size_t smem = (size_t)kAnyRows * 2 * head_dim * sizeof(float);
  hipStream_t s = (hipStream_t)stream;
#define SPV_ANY(QT) \
  hipLaunchKernelGGL(head_attn_any_kernel<QT>, dim3((unsigned)grid), dim3(64 * kAnyRows), smem, s, p, (int)groups)
  if (q_dtype == SPV_F32) SPV_ANY(SPV_F32);
  else if (q_dtype == SPV_BF16) SPV_ANY(SPV_BF16);
  else SPV_ANY(SPV_F16);
#undef SPV_ANY
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

}  // extern "C"
