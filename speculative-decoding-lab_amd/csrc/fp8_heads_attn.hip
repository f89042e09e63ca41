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
// verify chunks) times a range of steps of SK keys, its waves every eighth step.
// Everything stays transposed, so that no value changes lanes between the two
// products:
//   S^T = K Q^T: A = 16 keys x 32 dims, codes converted exactly (every e4m3 value
//     is a bf16 and an fp16 value) as they arrive from HBM, B = 16 rows, from LDS.
//     Lane (g, c) = (lane / 16, lane % 16) gets keys 4 g + i of each tile for row c.
//     The key that row r of tile t stands for is chosen, KG (r / 4) + 4 t + r % 4 of
//     the step, so that a lane's keys are KG = SK / 4 neighbours of one unit: one
//     block, one pair of scales.
//   O^T += V^T P^T: A = 16 dims x 32 keys, a lane's KG neighbours one 8- or 16-byte
//     load of a V^T row, B = the lane's own weights.
// The block's K scale multiplies the scores, its V scale the weights. The maximum of
// a row is raised (and O rescaled) only where a step passes it by more than 2^8.
// Roundings: scores, sums and O are fp32. A weight meets V in NP parts of bf16, 8
// bits each and of fp32's range (V's scale may be of any size): two for 16-bit
// queries (2^-17), three for fp32 ones. fp32 queries enter S in three parts.

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8, kTileThreads = 64 * kWaves;
constexpr int kGrid = 256;       // one workgroup per CU
constexpr int kMinSteps = 8;     // a piece has a step for each wave, where contexts are cut
constexpr float kLift = 8.f;     // log2 by which a step may pass the row's maximum
constexpr float kLowest = -3.402823466e38f;
constexpr int kCols = 32, kColPad = 4;  // dims of a combine pass

struct HeadPlan {  // host-chosen shape of a tiled call
  int RT, RG, SK, D, upb, equal;  // row tiles, row groups, keys of a step, units per block, pieces of equal length
  unsigned upb_magic;             // floor(2^32 / upb) + 1
  int aligned;                    // q and out on 16-byte addresses
  int* counters;                  // kGrid: arrivals of a segment's parts
  float* part;                    // slots of R x D sums and R x (maximum, sum)
};

template <int QT>
struct Parts {
  static constexpr int Q = QT == SPV_F32 ? 3 : 1, P = QT == SPV_F32 ? 3 : 2;
};

template <bool HI>
__device__ __forceinline__ uint32_t to_bf16x2(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t to_f16x2(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
}
// Eight codes as an operand.
template <bool F16>
__device__ __forceinline__ u32x4_t operand(uint32_t a, uint32_t b) {
  if constexpr (F16) return u32x4_t{to_f16x2<false>(a), to_f16x2<true>(a), to_f16x2<false>(b), to_f16x2<true>(b)};
  else return u32x4_t{to_bf16x2<false>(a), to_bf16x2<true>(a), to_bf16x2<false>(b), to_bf16x2<true>(b)};
}
template <bool F16>
__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}

// Keys that the rows of group rg of entry b see, and steps of them (one at least).
__device__ __forceinline__ int group_keys(const HeadAttn& p, int R, int start, int rg) {
  const int last = min(p.C - 1, (rg * R + R - 1) / p.ratio);
  return min(start + last + 1, p.max_ctx);
}
template <int SK>
__device__ __forceinline__ int group_steps(const HeadAttn& p, int R, int start, int rg) {
  return max(1, (group_keys(p, R, start, rg) + SK - 1) / SK);
}

template <int QT, int D, int RT, int SK>
__global__ __launch_bounds__(kTileThreads, 2) void head_attn_tile_kernel(HeadAttn p, HeadPlan pl) {
  constexpr bool F16 = QT == SPV_F16;
  constexpr int NQ = Parts<QT>::Q, NP = Parts<QT>::P, R = RT * 16, NCH = D / 32, NDT = D / 16, KT = SK / 16,
                KG = SK / 4, NM = KG / 8;
  constexpr int kQBytes = RT * NCH * NQ * 1024, kCombineBytes = kWaves * R * (kCols + kColPad) * 4;
  constexpr bool kQReg = RT * NCH * NQ <= 8;  // queries in registers, where they are few
  __shared__ __align__(16) uint8_t s_buf[kQBytes > kCombineBytes ? kQBytes : kCombineBytes];
  __shared__ float s_ml[2][kWaves][R];
  __shared__ float s_row[2][R];  // joined maximum and sum
  __shared__ int s_scan[kWaves], s_find[2], s_last;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;

  // ---- which piece: a number of steps (equal = 0: shares of all steps in a row) or of pieces per entry
  const int cpt = (p.B + kTileThreads - 1) / kTileThreads;  // entries of a thread
  const int b0 = min((int)threadIdx.x * cpt, p.B), b1 = min(b0 + cpt, p.B);
  auto per_entry = [&](int start, int P) {  // steps of an entry, or pieces of at most P of them
    int n = 0;
    for (int rg = 0; rg < pl.RG; ++rg) {
      const int k = group_steps<SK>(p, R, start, rg);
      n += P ? (k + P - 1) / P : k;
    }
    return n * p.Hkv;
  };
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int start = p.start[b];
    mine += per_entry(start, 0);
    if (blockIdx.x == 0) {
      const int sid = p.seq_ids[b];
      if (start < 0 || start + p.C > p.max_ctx || (p.lens && start + p.C > p.lens[sid])) flag_read(p, b);
    }
  }
  int total, before = block_exclusive_scan(mine, s_scan, &total);
  int P = (total + kGrid - 1) / kGrid;
  if (P < kMinSteps) P = kMinSteps;
  if (pl.equal) {
    while (true) {  // ends: with P the longest context, one piece per segment, of at most kGrid / 2 segments
      mine = 0;
      for (int b = b0; b < b1; ++b) mine += per_entry(p.start[b], P);
      before = block_exclusive_scan(mine, s_scan, &total);
      if (total <= kGrid) break;
      P += max(1, P >> 4);
    }
  }
  const int x0 = pl.equal ? (int)blockIdx.x : (int)blockIdx.x * P;
  const int x1 = min(total, pl.equal ? x0 + 1 : x0 + P);

  for (int cur = x0; cur < x1;) {
    __syncthreads();
    if (before <= cur && cur < before + mine) {
      int at = before;
      for (int b = b0; b < b1; ++b) {
        const int n = per_entry(p.start[b], pl.equal ? P : 0);
        if (cur < at + n) {
          s_find[0] = b;
          s_find[1] = cur - at;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
    const int b = __builtin_amdgcn_readfirstlane(s_find[0]);
    int off = __builtin_amdgcn_readfirstlane(s_find[1]);
    const int start = p.start[b], sid = p.seq_ids[b];
    int rg = 0, n = 0, k = 0;
    for (;; ++rg) {
      n = group_steps<SK>(p, R, start, rg);
      k = pl.equal ? (n + P - 1) / P : n;
      if (off < k * p.Hkv || rg == pl.RG - 1) break;
      off -= k * p.Hkv;
    }
    const int h = off / k, i_in = off - h * k;
    int first, last, nparts, my, slot0;  // steps [first, last); parts of the segment, which is this; slots
    if (pl.equal) {
      first = (int)((long long)n * i_in / k);
      last = (int)((long long)n * (i_in + 1) / k);
      nparts = k;
      my = i_in;
      slot0 = cur - i_in;
      cur = x1;
    } else {
      first = i_in;
      last = min(n, i_in + x1 - cur);
      const int s0 = cur - i_in;  // the segment's first step among all
      slot0 = s0;
      nparts = (s0 + n - 1) / P - s0 / P + 1;
      my = (int)blockIdx.x - s0 / P;
      cur += last - first;
    }
    // Slot of part i: its workgroup's first or second one (a share's first piece, or its last).
    auto slot_of = [&](int i) {
      if (pl.equal) return slot0 + i;
      const int wg = slot0 / P + i;
      return wg * P >= slot0 ? 2 * wg : 2 * wg + 1;
    };
    const int keys = group_keys(p, R, start, rg), units = max(1, (keys + 15) >> 4);
    const int rows = min(R, p.C * p.ratio - rg * R);
    const int32_t* const table = p.tables + (size_t)sid * p.maxb;
    const size_t page_bytes = (size_t)p.bs * D;
    const uint8_t* const kbase = p.kpool + ((size_t)p.layer * p.cap * p.Hkv + h) * page_bytes;
    const uint8_t* const vbase = p.vpool + ((size_t)p.layer * p.cap * p.Hkv + h) * page_bytes;
    const float* const sbase = p.scales + ((size_t)p.layer * p.Hkv + h) * p.cap * 2;
    const size_t block_bytes = page_bytes * p.Hkv;

    // ---- addresses of a step: the unit of the lane's K rows (of c) and of its own keys (of g)
    auto unit_at = [&](int step, int grp) { return min((step * SK + grp * KG) >> 4, units - 1); };
    auto block_id = [&](int u) {
      const int blk = pl.upb == 1 ? u : (int)__umulhi((unsigned)u, pl.upb_magic);
      return table[min(blk, p.maxb - 1)];
    };
    auto safe = [&](int id) {
      if ((unsigned)id < (unsigned)p.cap) return id;
      flag_read(p, b);
      return 0;
    };
    auto in_block = [&](int u) { return pl.upb == 1 ? 0 : (u - (int)__umulhi((unsigned)u, pl.upb_magic) * pl.upb) * 16; };
    auto kaddr = [&](int step, int id) {
      const int u = unit_at(step, c >> 2);
      const int tok = in_block(u) + (((step * SK + (c >> 2) * KG) & 15) + (c & 3));
      return kbase + (size_t)id * block_bytes + (size_t)(tok * D + 16 * g);
    };
    auto vaddr = [&](int step, int id) {
      const int u = unit_at(step, g);
      const int tok = in_block(u) + ((step * SK + g * KG) & 15);
      return vbase + (size_t)id * block_bytes + (size_t)(c * p.bs + tok);
    };
    u32x4_t kraw[KT][D / 64];
    uint32_t vraw[NDT][KG / 4];
    float2 sc;
    auto load_k = [&](const uint8_t* at, int t, int cc) {
      kraw[t][cc] = *reinterpret_cast<const u32x4_t*>(at + 4 * t * D + 64 * cc);
    };
    auto load_v = [&](const uint8_t* at, int dt) {
      if constexpr (KG == 16) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(at + (size_t)(dt * 16) * p.bs);
#pragma unroll
        for (int i = 0; i < 4; ++i) vraw[dt][i] = w[i];
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(at + (size_t)(dt * 16) * p.bs);
        vraw[dt][0] = w[0];
        vraw[dt][1] = w[1];
      }
    };
    auto load_scales = [&](int id) { sc = *reinterpret_cast<const float2*>(sbase + (size_t)id * 2); };
    int step = first + wave;
    int kid = 0, vid = 0;  // of the step after
    if (step < last) {
      const int k0 = block_id(unit_at(step, c >> 2)), v0 = block_id(unit_at(step, g));
      kid = block_id(unit_at(step + kWaves, c >> 2));
      vid = block_id(unit_at(step + kWaves, g));
      const uint8_t* const ka = kaddr(step, safe(k0));
      const uint8_t* const va = vaddr(step, safe(v0));
#pragma unroll
      for (int cc = 0; cc < D / 64; ++cc)
#pragma unroll
        for (int t = 0; t < KT; ++t) load_k(ka, t, cc);
      load_scales(safe(v0));
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) load_v(va, dt);
    }

    // ---- queries to LDS as operands: [part][row tile][chunk][lane] 16 bytes; dims of a chunk as K's bytes arrive
    for (int i = threadIdx.x; i < R * (D / 8); i += kTileThreads) {
      const int row = i / (D / 8), piece = i - row * (D / 8), r = rg * R + row;
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
        reinterpret_cast<u32x4_t*>(s_buf)[((q * RT + (row >> 4)) * NCH + ch) * 64 + ln] = w;
      }
    }
    __syncthreads();
    auto query = [&](int rt, int ch, int q) {
      return reinterpret_cast<const u32x4_t*>(s_buf)[((q * RT + rt) * NCH + ch) * 64 + lane];
    };
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
    int seen[RT];  // keys that the lane's row attends
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kLowest;
      l[rt] = 0.f;
      seen[rt] = min(start + min((rg * R + rt * 16 + c) / p.ratio, p.C - 1) + 1, p.max_ctx);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[rt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const int all_see = min(start + rg * R / p.ratio + 1, p.max_ctx);  // keys that every row attends
    const float factor = fabsf(p.scale_log2);

    auto run_step = [&](auto more_tag) {
      constexpr bool MORE = decltype(more_tag)::value;
      const bool masked = (step + 1) * SK > all_see;
      const float ksc = sc.x * factor, vsc = sc.y;
      const uint8_t *ka = nullptr, *va = nullptr;
      int vnext = 0;
      if constexpr (MORE) {
        ka = kaddr(step + kWaves, safe(kid));
        vnext = safe(vid);
        va = vaddr(step + kWaves, vnext);
        kid = block_id(unit_at(step + 2 * kWaves, c >> 2));
        vid = block_id(unit_at(step + 2 * kWaves, g));
      }
      f32x4_t s[RT][KT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int t = 0; t < KT; ++t) s[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        u32x4_t qv[RT][NQ];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if constexpr (kQReg) qv[rt][q] = qreg[rt][ch][q];
            else qv[rt][q] = query(rt, ch, q);
          }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const u32x4_t kop = operand<F16>(kraw[t][ch / 2][2 * (ch & 1)], kraw[t][ch / 2][2 * (ch & 1) + 1]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int q = NQ - 1; q >= 0; --q) s[rt][t] = mfma<F16>(kop, qv[rt][q], s[rt][t]);
        }
        if constexpr (MORE) {
          if (ch & 1) {
#pragma unroll
            for (int t = 0; t < KT; ++t) load_k(ka, t, ch / 2);
          }
        }
      }
      if constexpr (MORE) load_scales(vnext);
      const int base = step * SK + g * KG;  // the lane's first key
      uint32_t pw[RT][NM][NP][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float z[KT][4], top = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[t][i] = s[rt][t][i] * ksc;
        if (masked) {
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (base + 4 * t + i >= seen[rt]) z[t][i] = -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, z[t][i]);
        if (__any(top > m[rt] + kLift)) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float mn = fmaxf(m[rt], top), keep = __builtin_amdgcn_exp2f(m[rt] - mn);
          m[rt] = mn;
          l[rt] *= keep;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[rt][dt] *= keep;
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(z[t][i] - m[rt]);
            l[rt] += e;
            z[t][i] = e * vsc;
          }
#pragma unroll
          for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w = pack_bf16(z[t][2 * i], z[t][2 * i + 1]);
              pw[rt][t / 2][q][2 * (t & 1) + i] = w;
              if (q + 1 < NP) {
                z[t][2 * i] -= __uint_as_float(w << 16);
                z[t][2 * i + 1] -= __uint_as_float(w & 0xffff0000u);
              }
            }
        }
      }
      if (masked) {  // values behind the rows' last key are not looked at
        const int valid = keys - base;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int i = 0; i < KG / 4; ++i) {
            const int nb = min(max(valid - 4 * i, 0), 4);
            vraw[dt][i] &= nb == 4 ? 0xffffffffu : (1u << (8 * nb)) - 1u;
          }
        // A NaN among the chunk's own values reaches the rows that see it, and no other.
        uint32_t bad = 0;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int i = 0; i < KG / 4; ++i) bad |= ((vraw[dt][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (__any(bad != 0)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            u32x4_t sees[NM];
#pragma unroll
            for (int mm = 0; mm < NM; ++mm)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int key = base + 8 * mm + 2 * i;
                sees[mm][i] = (key < seen[rt] ? 0x3f80u : 0u) | (key + 1 < seen[rt] ? 0x3f800000u : 0u);
              }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
              f32x4_t count = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int mm = 0; mm < NM; ++mm) {
                u32x4_t is;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t w = ((vraw[dt][2 * mm + i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                  is[2 * i] = (w & 0x80u ? 0x3f80u : 0u) | (w & 0x8000u ? 0x3f800000u : 0u);
                  is[2 * i + 1] = (w & 0x800000u ? 0x3f80u : 0u) | (w & 0x80000000u ? 0x3f800000u : 0u);
                }
                count = mfma<false>(is, sees[mm], count);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (count[i] > 0.f) o[rt][dt][i] = __uint_as_float(0x7fc00000u);
            }
          }
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < KG / 4; ++i) {
              const uint32_t w = ((vraw[dt][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // NaN bytes
              vraw[dt][i] &= ~((w >> 7) * 0xffu);
            }
        }
      }
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        u32x4_t vop[NM];
#pragma unroll
        for (int mm = 0; mm < NM; ++mm) vop[mm] = operand<false>(vraw[dt][2 * mm], vraw[dt][2 * mm + 1]);
        if constexpr (MORE) load_v(va, dt);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int mm = 0; mm < NM; ++mm)
#pragma unroll
            for (int q = NP - 1; q >= 0; --q)
              o[rt][dt] = mfma<false>(vop[mm], u32x4_t{pw[rt][mm][q][0], pw[rt][mm][q][1], pw[rt][mm][q][2], pw[rt][mm][q][3]},
                                      o[rt][dt]);
      }
    };
    for (; step + kWaves < last; step += kWaves) run_step(std::true_type{});
    if (step < last) run_step(std::false_type{});

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
    __syncthreads();
    if ((int)threadIdx.x < R) {
      float mx = kLowest, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, s_ml[0][w][threadIdx.x]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        sum = fmaf(s_ml[1][w][threadIdx.x], __builtin_amdgcn_exp2f(s_ml[0][w][threadIdx.x] - mx), sum);
      s_row[0][threadIdx.x] = mx;
      s_row[1][threadIdx.x] = sum;
    }
    __syncthreads();
    const bool whole = nparts == 1;
    constexpr size_t kSlot = (size_t)R * (D + 2);  // floats of a slot
    float* const slot = pl.part + (whole ? 0 : (size_t)slot_of(my) * kSlot);
    const __amdgpu_buffer_rsrc_t slot_rsrc = coherent_rsrc(slot);
    // Four dims of a row, normalised, to the output.
    auto put = [&](int row, int e, f32x4_t v, float sum) {
      const int r = rg * R + row, j = r / p.ratio, hq = h * p.ratio + r - j * p.ratio;
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
    float* const s_o = reinterpret_cast<float*>(s_buf);  // [wave][row][kCols + pad]
    float keep[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) keep[rt] = __builtin_amdgcn_exp2f(m[rt] - s_row[0][rt * 16 + c]);
#pragma unroll
    for (int pass = 0; pass < D / kCols; ++pass) {
      if (pass) __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < kCols / 16; ++dt)
          *reinterpret_cast<f32x4_t*>(s_o + (wave * R + rt * 16 + c) * (kCols + kColPad) + dt * 16 + 4 * g) =
              o[rt][pass * (kCols / 16) + dt] * keep[rt];
      __syncthreads();
      for (int i = threadIdx.x; i < rows * (kCols / 4); i += kTileThreads) {
        const int row = i / (kCols / 4), e = (i - row * (kCols / 4)) * 4;
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          sum += *reinterpret_cast<const f32x4_t*>(s_o + (w * R + row) * (kCols + kColPad) + e);
        if (whole) put(row, pass * kCols + e, sum, s_row[1][row]);
        else store_coherent_b128(slot_rsrc, ((size_t)row * D + pass * kCols + e) * 4, __builtin_bit_cast(u32x4_t, sum));
      }
    }
    if (whole) continue;
    if ((int)threadIdx.x < R)
      store_coherent_b64(slot_rsrc, ((size_t)R * D + threadIdx.x * 2) * 4,
                         u32x2_t{__float_as_uint(s_row[0][threadIdx.x]), __float_as_uint(s_row[1][threadIdx.x])});
    // Counted at the workgroup in which the segment begins: it begins one segment at most that others go on with.
    if (!arrive_last(pl.counters + (pl.equal ? slot0 : slot0 / P), nparts, &s_last)) continue;

    // ---- the segment's last workgroup joins its parts, in their order
    for (int i = threadIdx.x; i < rows * (D / 4); i += kTileThreads) {
      const int row = i / (D / 4), e = (i - row * (D / 4)) * 4;
      float mx = kLowest, sum = 0.f;
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
      constexpr int kAt = 8;  // parts in flight
      for (int q0 = 0; q0 < nparts; q0 += kAt) {
        u32x4_t v[kAt];
        u32x2_t ml[kAt];
#pragma unroll
        for (int q = 0; q < kAt; ++q) {
          const __amdgpu_buffer_rsrc_t r = coherent_rsrc(pl.part + (size_t)slot_of(min(q0 + q, nparts - 1)) * kSlot);
          v[q] = load_coherent_b128(r, ((size_t)row * D + e) * 4);
          ml[q] = load_coherent_b64(r, ((size_t)R * D + row * 2) * 4);
        }
#pragma unroll
        for (int q = 0; q < kAt; ++q) {
          if (q0 + q >= nparts) break;
          const float mq = __uint_as_float(ml[q][0]), mn = fmaxf(mx, mq);
          const float was = __builtin_amdgcn_exp2f(mx - mn), is = __builtin_amdgcn_exp2f(mq - mn);
          mx = mn;
          sum = fmaf(__uint_as_float(ml[q][1]), is, sum * was);
          acc = acc * was + __builtin_bit_cast(f32x4_t, v[q]) * is;
        }
      }
      put(row, e, acc, sum);
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
  pl.RG = (int)((rows + 63) / 64);
  pl.RT = (int)(((rows + pl.RG - 1) / pl.RG + 15) / 16);
  pl.SK = d == 128 && pl.RT > 2 ? 32 : 64;
  pl.upb = bs / 16;
  pl.upb_magic = (unsigned)(0x100000000ULL / (unsigned)pl.upb + 1);
  const long long segs = (long long)B * pl.RG * Hkv, steps = ((long long)max_ctx + pl.SK - 1) / pl.SK;
  if (segs * steps > 0x3fffffffLL || ((long long)max_ctx / 16 + 1) * pl.upb > 0x7fffffffLL) return false;
  pl.equal = segs * 2 <= kGrid;
  return true;
}

constexpr size_t kCounterBytes = kGrid * sizeof(int);  // at the same place for calls of every shape
size_t tile_bytes(const HeadPlan& pl) {
  return kCounterBytes + (size_t)2 * kGrid * pl.RT * 16 * (pl.D + 2) * sizeof(float);
}

template <int QT, int D>
void launch_tile(const HeadAttn& p, const HeadPlan& pl, hipStream_t s) {
#define SPV_T(RT, SK) \
  hipLaunchKernelGGL((head_attn_tile_kernel<QT, D, RT, SK>), dim3(kGrid), dim3(kTileThreads), 0, s, p, pl)
  constexpr int kBig = D == 128 ? 32 : 64;
  if (pl.RT == 1) SPV_T(1, 64);
  else if (pl.RT == 2) SPV_T(2, 64);
  else if (pl.RT == 3) SPV_T(3, kBig);
  else SPV_T(4, kBig);
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
