// Attention of a batch whose sequences share long prefixes, over paged keys and
// values.
//
// Entry b's row j (q head hq, kv head hq / (Hq/Hkv)) attends, with
// softmax(scale * q.k), the first P_b positions of its prefix's sequence and
// then positions 0 .. start_b + j of its own. The softmax of the joined
// keys splits over key ranges: a range leaves, per row, m = max s, l = sum
// 2^(s - m) and o = sum 2^(s - m) v (s in log2 units), and ranges join by
// M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.
//
// So a prefix is walked once for all rows of all its entries: the rows of a
// group (entries with one prefix and one length) that share a kv head are laid
// end to end -- (member, chunk token, head of the group) -- and cut into tiles of
// 128. All (tile, 64 keys) units, laid end to end, are cut into equal shares, one
// per workgroup; a share's part of one tile is a segment and leaves a partial.
// An entry's own keys are walked by further workgroups, one per (entry, kv head,
// tile of its rows, range). A second launch joins each row's partials. Shares
// and segments are listed on the host (the prefixes and their lengths change
// when a request is admitted, not between rounds); the entries' own lengths are
// read on the device.
//
// Matrix path (bf16 queries over bf16 or fp8 pages, fp16 over fp16, head_dim 64
// or 128, 16-token blocks, a finite positive scale): a workgroup of four waves
// takes 128 rows, 32 per wave, and stages 64 keys at a time in LDS (two buffers),
// so a key read from the L2 once serves 128 rows. Per 16-key page and 16 rows
//   S^T = K Q^T    v_mfma_f32_16x16x32, A = 16 keys x 32 dims, B = Q^T fragments
//                  that stay in registers for the whole segment;
//   O^T += V^T P^T v_mfma_f32_16x16x32_f16 over two pages, P in fp16.
// S^T's accumulator layout is P^T's operand layout (lane l: keys 4 (l / 16) .. + 3
// of row l % 16), so the softmax moves no data between lanes. P in bf16 (8 bits)
// would miss the library's bf16 bar (2e-3 per sequence, of which rounding the
// output alone takes 1.7e-3); fp16 has 11 bits. bf16 values are staged as fp16
// times a power of two per segment, chosen from the first tile's largest |v|
// (which lands in [2^8, 2^9): every value from 2^-25 of it up is exact, a smaller
// one is off by at most 2^-33 of it); where a later value would pass fp16's range
// the segment runs again with the power from its largest |v|. fp8 codes are fp16
// values; a block's V scale, over the segment's largest, multiplies P.
#include <math.h>

#include <algorithm>
#include <map>
#include <utility>
#include <vector>

#include "spv_common.h"

using namespace spv;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The plan: a header, then the groups, their members (batch entries), each
// entry's place, the shares (first segment of each, and the end), the segments,
// and per (group, kv head, tile) its segments.
enum : int {
  PH_MAGIC = 0,
  PH_INTS,  // length of the plan
  PH_B,
  PH_C,
  PH_HQ,
  PH_HKV,
  PH_BS,
  PH_NG,    // groups
  PH_NSH,   // shares (a multiple of 8, or 0)
  PH_NSEG,  // segments
  PH_NT,    // (group, kv head, tile) triples
  PH_MAXP,  // longest prefix
  PH_GROUPS,
  PH_MEMBERS,
  PH_ENTRIES,
  PH_SHARES,
  PH_SEGS,
  PH_TILES,
  PH_WORDS
};
constexpr int kPlanMagic = 0x53505232;
enum : int { G_SID = 0, G_LEN, G_FIRST, G_COUNT, G_NT, G_TILE0, G_WORDS };  // G_NT: tiles of a kv head
enum : int { E_GROUP = 0, E_RANK, E_WORDS };
enum : int { S_GROUP = 0, S_HEAD, S_TILE, S_KEY0, S_KEY1, S_WORDS };
enum : int { T_SEG = 0, T_COUNT, T_WORDS };
constexpr int kTile = 128;  // rows
constexpr int kUnit = 64;   // keys

struct SharedParams {
  void* out;
  const void* q;
  const void* kpool;
  const void* vpool;
  const float* scales;
  const int32_t* tables;
  const int32_t* seq_ids;
  const int32_t* start;
  const int32_t* lens;
  int32_t* ctr;
  const int32_t* plan;
  float* part_o;   // partial rows x d
  float* part_ml;  // partial rows x 2
  int maxb, B, C, Hq, Hkv, ratio, G, d, bs, layer, cap;
  int shares;              // workgroups that walk prefixes
  int own_range, own_max;  // keys per own range (a multiple of the block size), ranges per entry at most
  int own_tiles;           // tiles of an entry's rows
  int max_ctx;
  long long own_part;      // first partial row of the own ranges
  float scale_log2;
};

// One piece of work: rows [row0, row0 + rows) of a group's (or one entry's) row
// order over keys [key0, key1) of one sequence.
struct Item {
  int group, sid, b, h, row0, rows, key0, key1, first, limit;  // limit: row j sees keys <= limit + j (an entry's own)
  long long part;                                                // its first partial row
};

__device__ __forceinline__ void flag_bad_read(const SharedParams& p, int b) {
  if (p.ctr) p.ctr[CTR_BAD_READ] = b + 1;
}

__device__ __forceinline__ void segment_item(const SharedParams& p, int seg, Item& it) {
  const int32_t* s = p.plan + p.plan[PH_SEGS] + (size_t)seg * S_WORDS;
  const int32_t* g = p.plan + p.plan[PH_GROUPS] + (size_t)s[S_GROUP] * G_WORDS;
  it.group = s[S_GROUP];
  it.sid = g[G_SID];
  it.h = s[S_HEAD];
  it.first = p.plan[PH_MEMBERS] + g[G_FIRST];
  it.b = p.plan[it.first];
  it.row0 = s[S_TILE] * kTile;
  it.rows = min(kTile, g[G_COUNT] * p.G - it.row0);
  it.key0 = s[S_KEY0];
  it.key1 = s[S_KEY1];
  it.limit = 0x3fffffff;
  it.part = (long long)seg * kTile;
  if (threadIdx.x == 0 && p.lens && p.lens[it.sid] < g[G_LEN]) flag_bad_read(p, it.b);
}

// Own work `o`: false where the range has no keys.
__device__ __forceinline__ bool own_item(const SharedParams& p, int o, Item& it) {
  const int s = o % p.own_max, bht = o / p.own_max, t = bht % p.own_tiles, bh = bht / p.own_tiles;
  it.group = -1;
  it.b = bh / p.Hkv;
  it.h = bh - it.b * p.Hkv;
  it.sid = p.seq_ids[it.b];
  it.limit = p.start[it.b];
  const int L = it.limit + p.C, seen = min(max(L, 0), p.max_ctx);
  if (threadIdx.x == 0 && s == 0 && it.h == 0 && (it.limit < 0 || L > p.max_ctx || (p.lens && p.lens[it.sid] < L)))
    flag_bad_read(p, it.b);
  it.row0 = t * kTile;
  it.rows = min(kTile, p.G - it.row0);
  it.first = 0;
  it.key0 = s * p.own_range;
  it.key1 = min(it.key0 + p.own_range, seen);
  it.part = p.own_part + ((long long)bh * p.own_max + s) * p.G + it.row0;
  return it.key0 < it.key1;
}

// The share of workgroup `id`: workgroups go round-robin over the 8 XCDs, each of
// which takes an eighth of the shares in a row -- of one kv head, if there are few --
// so that its L2 serves one stretch of keys to all of its workgroups.
__device__ __forceinline__ int share_of(const SharedParams& p, int id) { return (id & 7) * (p.shares >> 3) + (id >> 3); }

// Row R of an item's row order: its entry, chunk token and q head.
__device__ __forceinline__ void row_at(const SharedParams& p, const Item& it, int R, int& b, int& j, int& hq) {
  int r = R;
  b = it.b;
  if (it.group >= 0) {
    const int m = R / p.G;
    r = R - m * p.G;
    b = p.plan[it.first + m];
  }
  j = r / p.ratio;
  hq = it.h * p.ratio + (r - j * p.ratio);
}

__device__ __forceinline__ int block_of(const SharedParams& p, const Item& it, int pos) {
  const int phys = p.tables[(size_t)it.sid * p.maxb + pos / p.bs];
  if ((unsigned)phys < (unsigned)p.cap) return phys;
  flag_bad_read(p, it.b);
  return 0;
}

// ------------------------------------------------------------------ any shape
// fp32 arithmetic in LDS tiles of 64 rows and 16 keys; any types, head_dim up to
// 256, any block size. Row j of a chunk adds only the keys it sees, so what
// later positions hold (infinities, NaN) never reaches it. Four threads per row,
// each every fourth dim.
constexpr int kThreads = 256;
constexpr int kRows = 64;
constexpr int kKeys = 16;
constexpr int kMaxD = 256;
__host__ __device__ constexpr size_t valu_lds(int d) {
  return (size_t)((kRows + 2 * kKeys) * (d + 1) + kRows * (kKeys + 1) + 2 * kRows) * sizeof(float);
}

// MD: a bound on head_dim.
template <int QT, int KT, int MD>
__device__ __forceinline__ void valu_item(const SharedParams& p, const Item& it, float* smem) {
  const int d = p.d, pitch = d + 1;
  float* Qs = smem;                    // [64][d], in log2 units
  float* Ks = Qs + kRows * pitch;      // [16][d]
  float* Vs = Ks + kKeys * pitch;      // [16][d]
  float* Ps = Vs + kKeys * pitch;      // [64][17]
  float* As = Ps + kRows * (kKeys + 1);
  int* Lim = reinterpret_cast<int*>(As + kRows);  // last key a row sees
  const int row = threadIdx.x >> 2, part = threadIdx.x & 3;
#pragma unroll 1
  for (int r0 = 0; r0 < it.rows; r0 += kRows) {
    const int nr = min(kRows, it.rows - r0);
#pragma unroll 1
    for (int i = threadIdx.x; i < nr * d; i += kThreads) {
      const int rr = i / d, e = i - rr * d;
      int b, j, hq;
      row_at(p, it, it.row0 + r0 + rr, b, j, hq);
      Qs[rr * pitch + e] = load_elem<QT>(p.q, (((size_t)b * p.C + j) * p.Hq + hq) * d + e) * p.scale_log2;
      if (e == 0) Lim[rr] = it.group >= 0 ? it.limit : it.limit + j;
    }
    float m = -INFINITY, l = 0.f;  // of row threadIdx.x, kept by the first 64 threads
    float o[MD / 4];               // dims part, part + 4, ... of row `row`
#pragma unroll
    for (int k = 0; k < MD / 4; ++k) o[k] = 0.f;
    __syncthreads();
#pragma unroll 1
    for (int t0 = it.key0; t0 < it.key1; t0 += kKeys) {
      const int nt = min(kKeys, it.key1 - t0);
#pragma unroll 1
      for (int i = threadIdx.x; i < nt * d; i += kThreads) {
        const int tt = i / d, e = i - tt * d;
        const int pos = t0 + tt, phys = block_of(p, it, pos), off = pos % p.bs;
        const size_t slot = ((size_t)p.layer * p.cap + phys) * p.Hkv + it.h;
        float kv = load_elem<KT>(p.kpool, (slot * p.bs + off) * d + e);
        float vv = load_elem<KT>(p.vpool, (slot * d + e) * p.bs + off);
        if constexpr (KT == SPV_FP8E4M3) {
          const float* sc = p.scales + ((size_t)p.layer * p.cap + phys) * 2;
          kv *= sc[0];
          vv *= sc[1];
        }
        Ks[tt * pitch + e] = kv;
        Vs[tt * pitch + e] = vv;
      }
      __syncthreads();
#pragma unroll 1
      for (int i = threadIdx.x; i < nr * kKeys; i += kThreads) {
        const int rr = i / kKeys, tt = i - rr * kKeys;
        float sc = -INFINITY;
        if (tt < nt && t0 + tt <= Lim[rr]) {
          sc = 0.f;
          for (int e = 0; e < d; ++e) sc = fmaf(Qs[rr * pitch + e], Ks[tt * pitch + e], sc);
        }
        Ps[rr * (kKeys + 1) + tt] = sc;
      }
      __syncthreads();
      if ((int)threadIdx.x < nr) {
        float* P = Ps + threadIdx.x * (kKeys + 1);
        float mx = m;
        for (int tt = 0; tt < kKeys; ++tt) mx = fmaxf(mx, P[tt]);
        const float ref = mx == -INFINITY ? 0.f : mx;  // a row without a finite score yet: its P are 0 (or NaN)
        const float alpha = exp2f(m - ref);
        float sum = 0.f;
        for (int tt = 0; tt < kKeys; ++tt) {
          P[tt] = exp2f(P[tt] - ref);
          sum += P[tt];
        }
        l = l * alpha + sum;
        m = mx;
        As[threadIdx.x] = alpha;
      }
      __syncthreads();
      if (row < nr) {
        const float alpha = As[row];
        const int n = min(nt, Lim[row] - t0 + 1);
#pragma unroll
        for (int k = 0; k < MD / 4; ++k) o[k] *= alpha;
#pragma unroll 1
        for (int tt = 0; tt < n; ++tt) {
          const float pr = Ps[row * (kKeys + 1) + tt];
          const float* v = Vs + tt * pitch + part;
#pragma unroll
          for (int k = 0; k < MD / 4; ++k)
            if (part + 4 * k < d) o[k] = fmaf(pr, v[4 * k], o[k]);
        }
      }
      __syncthreads();
    }
    float* const out = p.part_o + (size_t)(it.part + r0 + row) * d + part;
    if (row < nr) {
#pragma unroll
      for (int k = 0; k < MD / 4; ++k)
        if (part + 4 * k < d) out[4 * k] = o[k];
    }
    if ((int)threadIdx.x < nr)
      *reinterpret_cast<float2*>(&p.part_ml[(size_t)(it.part + r0 + threadIdx.x) * 2]) = make_float2(m, l);
    __syncthreads();
  }
}

// Workgroups [0, shares) walk prefixes, the others entries' own keys.
template <typename F>
__device__ __forceinline__ void for_items(const SharedParams& p, F&& run) {
  const int id = blockIdx.x;
  int s = 0, end = 1;
  if (id < p.shares) {
    const int32_t* sh = p.plan + p.plan[PH_SHARES] + share_of(p, id);
    s = sh[0];
    end = sh[1];
  }
#pragma unroll 1
  for (; s < end; ++s) {
    Item it;
    if (id < p.shares) segment_item(p, s, it);
    else if (!own_item(p, id - p.shares, it)) return;
    run(it);
  }
}

template <int QT, int KT>
__global__ __launch_bounds__(kThreads) void shared_valu_kernel(SharedParams p) {
  extern __shared__ float smem[];
  for_items(p, [&](const Item& it) { valu_item<QT, KT, kMaxD>(p, it, smem); });
}

// -------------------------------------------------------------- matrix kernels
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// A row's scores may exceed its reference maximum by this much (log2 units) before
// its sums are rescaled: P stays below 2^8, far inside fp16.
constexpr float kSlack = 8.f;

__device__ __forceinline__ uint32_t pack2_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}
// v_max3_f32 on matrix results (fmaxf would first canonicalise each input).
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
// Running maximum of the absolute values (as bits) of two 16-bit floats a word.
__device__ __forceinline__ uint32_t max_abs2(uint32_t w, uint32_t m) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, w & 0x7fff7fffu),
                                                                __builtin_bit_cast(u16x2_t, m)));
}
// The staging power for a largest finite |v| of mx: mx 2^k in [2^8, 2^9), 0 where all are zero.
__device__ __forceinline__ int stage_exponent(float mx) {
  if (!(mx > 0.f)) return 0;
  int e;
  frexpf(mx, &e);
  return min(126, max(-126, 9 - e));
}

template <int D, int KT>
struct Lds {
  // 32 bytes of padding on a K row and a V^T row: their 16-byte reads meet no bank twice.
  static constexpr int KP = D + 16, VP = kUnit + 16;
  static constexpr int kK = kUnit * KP, kV = D * VP;              // elements of a buffer
  static constexpr size_t kBytes = 2 * (size_t)(kK + kV) * 2 + 64;  // two of each, and a word per wave
};

template <int D, int KT>
__global__ __launch_bounds__(kThreads, 2) void shared_mfma_kernel(SharedParams p) {
  constexpr bool kF16 = KT == SPV_F16, kFp8 = KT == SPV_FP8E4M3;
  constexpr int QT = kF16 ? SPV_F16 : SPV_BF16;
  constexpr int ES = kFp8 ? 1 : 2;
  constexpr int KS = D / 32, MT = D / 16, NT = 2;
  using LD = Lds<D, KT>;
  constexpr int KP = LD::KP, VP = LD::VP;
  static_assert(valu_lds(D) <= LD::kBytes, "the any-shape walk reuses this memory");
  __shared__ __align__(16) uint8_t smem[LD::kBytes];
  uint16_t* const sK = reinterpret_cast<uint16_t*>(smem);
  uint16_t* const sV = sK + 2 * LD::kK;
  uint32_t* const sMax = reinterpret_cast<uint32_t*>(sV + 2 * LD::kV);

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, g = lane >> 4;
  const float sl2 = p.scale_log2, inv_sl2 = 1.f / p.scale_log2;
  const f16x2_t ones = f16x2_t{(_Float16)1.f, (_Float16)1.f};

  auto wg_max = [&](uint32_t m) {  // the workgroup's largest m, in every thread
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    __syncthreads();
    if (lane == 0) sMax[w] = m;
    __syncthreads();
    return max(max(sMax[0], sMax[1]), max(sMax[2], sMax[3]));
  };

  for_items(p, [&](const Item& it) {
    // This lane's rows (columns of S^T): 16 nt + i16 of the wave's 32.
    int lim[NT];
    bool valid[NT];
    uint4 qf[NT][KS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int R = w * 32 + nt * 16 + i16;
      valid[nt] = R < it.rows;
      int b, j, hq;
      row_at(p, it, it.row0 + min(R, it.rows - 1), b, j, hq);
      lim[nt] = it.group >= 0 ? it.limit : it.limit + j;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + (((size_t)b * p.C + j) * p.Hq + hq) * D + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[nt][ks] = *reinterpret_cast<const uint4*>(q + 32 * ks);
    }
    const bool active = w * 32 < it.rows;
    const int h = __builtin_amdgcn_readfirstlane(it.h), key0 = __builtin_amdgcn_readfirstlane(it.key0),
              key1 = __builtin_amdgcn_readfirstlane(it.key1), own0 = __builtin_amdgcn_readfirstlane(it.limit);
    const int pages = (key1 - key0 + 15) >> 4, ntiles = (key1 - key0 + kUnit - 1) / kUnit;
    const int32_t* table = p.tables + (size_t)__builtin_amdgcn_readfirstlane(it.sid) * p.maxb + (key0 >> 4);

    // Block ids (and an fp8 page's scales) of 64 pages in the lanes of a register;
    // pages past the range repeat its last one.
    int ids = 0;
    float ksc = 1.f, vsc = 1.f;
    float vref = 1.f;  // fp8: the range's largest V scale
    auto page_ids = [&](int first) {
      const int phys = table[min(first + lane, pages - 1)];
      if ((unsigned)phys >= (unsigned)p.cap) flag_bad_read(p, it.b);
      return (unsigned)phys < (unsigned)p.cap ? phys : 0;
    };
    auto scales_of = [&](int phys) {
      return *reinterpret_cast<const float2*>(p.scales + ((size_t)p.layer * p.cap + phys) * 2);
    };
    auto window = [&](int first) {
      ids = page_ids(first);
      if constexpr (kFp8) {
        const float2 s = scales_of(ids);
        ksc = s.x;
        vsc = vref > 0.f ? s.y / vref : 0.f;
      }
    };

    // Staging. K: 16-byte pieces of a page in memory order. V: (dim, page pair,
    // half) items: 8 keys of the even and 8 of the odd page. In a V^T row key 4 gg +
    // j of page 2 q + hh sits at 32 q + 8 gg + 4 hh + j, so that lane group gg's
    // 16-byte read holds its keys of both pages.
    constexpr int kKN = kUnit * D * ES / 16 / kThreads;  // K pieces per thread
    constexpr int kVN = 4 * D / kThreads;                // V items per thread
    struct Stage {
      u32x4_t k[kKN];
      u32x4_t v[kVN][2];  // fp8: the first 8 bytes
    };
    const size_t layer_base = (size_t)p.layer * p.cap;
    auto page = [&](const void* pool, int phys) {
      return static_cast<const uint8_t*>(pool) + ((layer_base + phys) * p.Hkv + h) * (size_t)(16 * D * ES);
    };
    constexpr int kPer = D * ES;  // 16-byte pieces of a page
    auto load = [&](Stage& S, int t) {
#pragma unroll
      for (int i = 0; i < kKN; ++i) {
        const int pi = (w * 64 + i * kThreads) / kPer, c = (tid + i * kThreads) % kPer;
        const int phys = __builtin_amdgcn_readlane(ids, (4 * t + pi) & 63);
        S.k[i] = *reinterpret_cast<const u32x4_t*>(page(p.kpool, phys) + 16 * c);
      }
#pragma unroll
      for (int i = 0; i < kVN; ++i) {
        const int q = (w * 64 + i * kThreads) / (2 * D), c = (tid + i * kThreads) % (2 * D);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int phys = __builtin_amdgcn_readlane(ids, (4 * t + 2 * q + hh) & 63);
          const uint8_t* v = page(p.vpool, phys) + 8 * ES * c;
          if constexpr (kFp8) {
            const uint2 x = *reinterpret_cast<const uint2*>(v);
            S.v[i][hh] = u32x4_t{x.x, x.y, 0u, 0u};
          } else {
            S.v[i][hh] = *reinterpret_cast<const u32x4_t*>(v);
          }
        }
      }
    };
    float vs = 1.f;          // bf16: the staging factor 2^vk
    int vk = 0;
    uint32_t vmax = 0;       // bf16: largest |v| bits staged (both halves)
    bool dirty = false;      // a value that some row of the tile may not see is not finite
    // Zeroes the values of keys past the range's end, and looks for non-finite ones
    // among the chunk's own keys, which earlier rows do not see: P = 0 would not
    // keep them out of a product.
    auto edge = [&](Stage& S, int t) {
      const int t0 = key0 + t * kUnit;
      if (t0 + kUnit <= key1 && (it.group >= 0 || t0 + kUnit - 1 <= own0)) return;
#pragma unroll
      for (int i = 0; i < kVN; ++i) {
        const int idx = tid + i * kThreads, q = idx / (2 * D), half = idx & 1;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          u32x4_t x = S.v[i][hh];
          const int k0 = t0 + 32 * q + 16 * hh + 8 * half;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            constexpr uint32_t kMask = kFp8 ? 0xffu : 0xffffu;
            const int word = e * ES / 4, shift = 8 * (e * ES % 4);
            const uint32_t bits = (x[word] >> shift) & kMask;
            const bool bad = kFp8 ? (bits & 0x7fu) == 0x7fu
                                  : (kF16 ? (bits & 0x7c00u) == 0x7c00u : (bits & 0x7f80u) == 0x7f80u);
            if (k0 + e >= key1) x[word] &= ~(kMask << shift);
            else dirty |= bad && k0 + e > own0;
          }
          S.v[i][hh] = x;
        }
      }
    };
    auto store = [&](Stage& S, int t, int buf) {
      edge(S, t);
      uint16_t* const K = sK + buf * LD::kK;
      uint16_t* const V = sV + buf * LD::kV;
#pragma unroll
      for (int i = 0; i < kKN; ++i) {
        const int pi = (w * 64 + i * kThreads) / kPer, c = (tid + i * kThreads) % kPer;
        if constexpr (kFp8) {  // 16 codes: bf16 values, exactly
          const int key = 16 * pi + c / (D / 16), col = c % (D / 16);
          const u32x4_t x = S.k[i];
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[e], 1.f, false));
            y[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[e], 1.f, true));
          }
          *reinterpret_cast<uint4*>(&K[key * KP + 16 * col]) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(&K[key * KP + 16 * col + 8]) = make_uint4(y[4], y[5], y[6], y[7]);
        } else {
          const int key = 16 * pi + c / (D / 8), col = c % (D / 8);
          *reinterpret_cast<u32x4_t*>(&K[key * KP + 8 * col]) = S.k[i];
        }
      }
#pragma unroll
      for (int i = 0; i < kVN; ++i) {
        const int idx = tid + i * kThreads, q = idx / (2 * D), dim = (idx >> 1) % D, half = idx & 1;
        uint2 y[2][2];  // [page][keys 0-3, 4-7 of the half]
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const u32x4_t x = S.v[i][hh];
          if constexpr (kF16) {
            y[hh][0] = make_uint2(x[0], x[1]);
            y[hh][1] = make_uint2(x[2], x[3]);
          } else if constexpr (kFp8) {
            uint32_t z[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              z[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[e], 1.f, false));
              z[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[e], 1.f, true));
            }
            y[hh][0] = make_uint2(z[0], z[1]);
            y[hh][1] = make_uint2(z[2], z[3]);
          } else {
            uint32_t z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              vmax = max_abs2(x[e], vmax);
              z[e] = pack2_f16(__uint_as_float(x[e] << 16) * vs, __uint_as_float(x[e] & 0xffff0000u) * vs);
            }
            y[hh][0] = make_uint2(z[0], z[1]);
            y[hh][1] = make_uint2(z[2], z[3]);
          }
        }
        uint16_t* const row = &V[dim * VP + 32 * q + 16 * half];
        *reinterpret_cast<uint4*>(row) = make_uint4(y[0][0].x, y[0][0].y, y[1][0].x, y[1][0].y);
        *reinterpret_cast<uint4*>(row + 8) = make_uint4(y[0][1].x, y[0][1].y, y[1][1].x, y[1][1].y);
      }
    };

    f32x4_t o[MT][NT];
    float m[NT], l[NT], thr[NT];  // thr: the score above which m must grow
    bool again = false;
    if constexpr (kFp8) {
      float mx = 0.f;
      for (int pg = tid; pg < pages; pg += kThreads) {
        const int phys = table[pg];
        if ((unsigned)phys < (unsigned)p.cap) mx = fmaxf(mx, scales_of(phys).y);
      }
      vref = __uint_as_float(wg_max(__float_as_uint(mx)));
    }
    for (int attempt = 0;; ++attempt) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[mt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = 0.f;
        thr[nt] = -INFINITY;
      }
      Stage S;
      window(0);
      load(S, 0);
      if constexpr (!kF16 && !kFp8) {
        // The largest finite |v| of the first tile, or (again) of the whole range.
        uint32_t mx = 0;
        auto take = [&](const Stage& X) {
#pragma unroll
          for (int i = 0; i < kVN; ++i)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const u32x4_t x = X.v[i][hh];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t lo = x[e] & 0x7fffu, hi = (x[e] >> 16) & 0x7fffu;
                if (lo < 0x7f80u) mx = max(mx, lo);
                if (hi < 0x7f80u) mx = max(mx, hi);
              }
            }
        };
        edge(S, 0);
        take(S);
        if (again) {
          for (int t = 1; t < ntiles; ++t) {
            if ((t & 15) == 0) window(4 * t);
            load(S, t);
            edge(S, t);
            take(S);
          }
          window(0);
          load(S, 0);
        }
        vk = stage_exponent(__uint_as_float(wg_max(mx) << 16));
        vs = ldexpf(1.f, vk);
        vmax = 0;
      }
      float ksn = ksc, vsn = vsc;  // the scales of the tile in the stage
      store(S, 0, 0);
      if (ntiles > 1) load(S, 1);
      __syncthreads();
      for (int t = 0; t < ntiles; ++t) {
        const float ks_t = ksn, vs_t = vsn;
        if (t + 1 < ntiles) {
          store(S, t + 1, (t + 1) & 1);
          if (((t + 2) & 15) == 0 && t + 2 < ntiles) window(4 * (t + 2));
          if (t + 2 < ntiles) load(S, t + 2);
        }
        if ((t & 15) == 15) ksn = ksc, vsn = vsc;
        if (active) {
          const uint16_t* K = sK + (t & 1) * LD::kK;
          const uint16_t* V = sV + (t & 1) * LD::kV;
          f32x4_t sc[4][NT];
#pragma unroll
          for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[kt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const uint4 kf = *reinterpret_cast<const uint4*>(&K[(16 * kt + i16) * KP + 32 * ks + 8 * g]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                sc[kt][nt] = kF16 ? __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, kf),
                                                                            __builtin_bit_cast(f16x8_t, qf[nt][ks]),
                                                                            sc[kt][nt], 0, 0, 0)
                                  : __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf),
                                                                             __builtin_bit_cast(bf16x8_t, qf[nt][ks]),
                                                                             sc[kt][nt], 0, 0, 0);
            }
          }
          if constexpr (kFp8) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
              const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_t), (4 * t + kt) & 63));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) sc[kt][nt] *= f;
            }
          }
          const int t0 = key0 + t * kUnit;
          if (t0 + kUnit > key1 || (it.group < 0 && t0 + kUnit - 1 > own0)) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                  const int key = t0 + 16 * kt + 4 * g + jj;
                  if (key >= key1 || key > lim[nt]) sc[kt][nt][jj] = -INFINITY;
                }
          }
          float mx[NT];
          bool grow = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float a0 = max3_raw(sc[0][nt][0], sc[0][nt][1], sc[0][nt][2]);
            float a1 = max3_raw(sc[0][nt][3], sc[1][nt][0], sc[1][nt][1]);
            float a2 = max3_raw(sc[1][nt][2], sc[1][nt][3], sc[2][nt][0]);
            float a3 = max3_raw(sc[2][nt][1], sc[2][nt][2], sc[2][nt][3]);
            float a4 = max3_raw(sc[3][nt][0], sc[3][nt][1], sc[3][nt][2]);
            a0 = max3_raw(a0, a1, a2);
            a3 = max3_raw(a3, a4, sc[3][nt][3]);
            mx[nt] = fmaxf(a0, a3);
            grow |= mx[nt] > thr[nt];
          }
          if (__any(grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float a = fmaxf(mx[nt], __shfl_xor(mx[nt], 16, 64));
              a = fmaxf(a, __shfl_xor(a, 32, 64));
              const float m_new = fmaxf(m[nt], a * sl2);
              const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nt] - m_new);
              l[nt] *= alpha;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) o[mt][nt] *= alpha;
              m[nt] = m_new;
              thr[nt] = (m_new + kSlack) * inv_sl2;
            }
          }
          uint32_t ph[2][NT][4];
#pragma unroll
          for (int kt = 0; kt < 4; ++kt) {
            float f = 1.f;
            if constexpr (kFp8)
              f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_t), (4 * t + kt) & 63));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float mu = m[nt] == -INFINITY ? 0.f : m[nt];
              float e[4];
#pragma unroll
              for (int jj = 0; jj < 4; ++jj) e[jj] = __builtin_amdgcn_exp2f(fmaf(sc[kt][nt][jj], sl2, -mu));
              if constexpr (kFp8) {
                l[nt] += (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) e[jj] *= f;
              }
              const uint32_t p01 = pack2_f16(e[0], e[1]), p23 = pack2_f16(e[2], e[3]);
              ph[kt >> 1][nt][2 * (kt & 1)] = p01;
              ph[kt >> 1][nt][2 * (kt & 1) + 1] = p23;
              if constexpr (!kFp8) {  // the sum takes P as it enters P V
                l[nt] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p01), ones, l[nt], false);
                l[nt] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p23), ones, l[nt], false);
              }
            }
          }
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const f16x8_t va = __builtin_bit_cast(
                  f16x8_t, *reinterpret_cast<const uint4*>(&V[(16 * mt + i16) * VP + 32 * q + 8 * g]));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                o[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    va, __builtin_bit_cast(f16x8_t, make_uint4(ph[q][nt][0], ph[q][nt][1], ph[q][nt][2], ph[q][nt][3])),
                    o[mt][nt], 0, 0, 0);
            }
        }
        __syncthreads();
      }
      if constexpr (kF16 || kFp8) break;
      if (attempt == 1) break;
      // bits of the largest |v| that stays within fp16 at this power
      const uint32_t top = min(__float_as_uint(ldexpf(65504.f, -vk)) >> 16, 0x7f7fu);
      again = __syncthreads_or((vmax & 0xffffu) > top || (vmax >> 16) > top);
      if (!again) break;
    }
    if (it.group < 0 && __syncthreads_or(dirty)) {
      valu_item<QT, KT, D>(p, it, reinterpret_cast<float*>(smem));
      return;
    }
    const float post = kFp8 ? vref : ldexpf(1.f, -vk);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] += __shfl_xor(l[nt], 16, 64);
      l[nt] += __shfl_xor(l[nt], 32, 64);
      if (!valid[nt]) continue;
      const size_t row = (size_t)(it.part + w * 32 + nt * 16 + i16);
      if (g == 0) *reinterpret_cast<float2*>(&p.part_ml[row * 2]) = make_float2(m[nt], l[nt]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        *reinterpret_cast<f32x4_t*>(&p.part_o[row * D + 16 * mt + 4 * g]) = o[mt][nt] * post;
    }
  });
}

// ----------------------------------------------------------------------- join
// LPR lanes per (entry, chunk token, q head): four consecutive dims per lane (VEC,
// head_dim = 4 LPR), or dims lane + 64 k of any head_dim up to 256. The row's
// partials, the prefix's segments in key order and then its own ranges, are added
// in that order whatever finished first.
template <int QT, int LPR, bool VEC>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(SharedParams p) {
  const int lane = threadIdx.x % LPR;
  const long long row = (long long)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  if (row >= (long long)p.B * p.C * p.Hq) return;
  const int hq = (int)(row % p.Hq), bj = (int)(row / p.Hq), b = bj / p.C, j = bj - b * p.C;
  const int h = hq / p.ratio, r = j * p.ratio + (hq - h * p.ratio);
  const int32_t* e = p.plan + p.plan[PH_ENTRIES] + (size_t)b * E_WORDS;
  int np = 0;
  long long pre = 0;  // the prefix's partial row of segment 0
  if (e[E_GROUP] >= 0) {
    const int32_t* g = p.plan + p.plan[PH_GROUPS] + (size_t)e[E_GROUP] * G_WORDS;
    const long long R = (long long)e[E_RANK] * p.G + r;
    const int32_t* t = p.plan + p.plan[PH_TILES] + (size_t)(g[G_TILE0] + h * g[G_NT] + (int)(R / kTile)) * T_WORDS;
    np = t[T_COUNT];
    pre = (long long)t[T_SEG] * kTile + R % kTile;
  }
  const int seen = min(max(p.start[b] + p.C, 0), p.max_ctx);
  const int n = np + (seen + p.own_range - 1) / p.own_range;
  const long long own = p.own_part + (long long)(b * p.Hkv + h) * p.own_max * p.G + r;
  auto part = [&](int s) { return (size_t)(s < np ? pre + (long long)s * kTile : own + (long long)(s - np) * p.G); };
  float M = -INFINITY;
  for (int s = lane; s < n; s += LPR) M = fmaxf(M, p.part_ml[part(s) * 2]);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, LPR));
  const float ref = M == -INFINITY ? 0.f : M;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, L = 0.f;
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const size_t at = part(s);
    const float2 ml = *reinterpret_cast<const float2*>(&p.part_ml[at * 2]);
    const float w = exp2f(ml.x - ref);
    L += w * ml.y;
    const float* o = p.part_o + at * p.d;
    if constexpr (VEC) {
      const float4 x = *reinterpret_cast<const float4*>(o + 4 * lane);
      acc[0] += w * x.x;
      acc[1] += w * x.y;
      acc[2] += w * x.z;
      acc[3] += w * x.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < p.d) acc[k] += w * o[lane + 64 * k];
    }
  }
  const float inv = 1.f / L;
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[k] *= inv;
  const size_t at = (size_t)row * p.d;
  if constexpr (!VEC) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane + 64 * k < p.d) store_elem<QT>(p.out, at + lane + 64 * k, acc[k]);
  } else if constexpr (QT == SPV_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + 4 * lane) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w[k] = QT == SPV_BF16 ? f32_to_bf16(acc[2 * k]) | (uint32_t)f32_to_bf16(acc[2 * k + 1]) << 16
                            : f32_to_f16(acc[2 * k]) | (uint32_t)f32_to_f16(acc[2 * k + 1]) << 16;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at + 4 * lane) = make_uint2(w[0], w[1]);
  }
}

// ----------------------------------------------------------------------- plan
struct Group {
  int sid, len;
  std::vector<int> members;
};

int make_plan(std::vector<int32_t>& plan, const int32_t* ids, const int32_t* lens, int B, int C, int Hq, int Hkv,
              int bs) {
  const long long G = (long long)C * (Hq / Hkv);
  std::vector<Group> groups;
  std::map<std::pair<int32_t, int32_t>, size_t> index;
  std::vector<int32_t> entries(E_WORDS * (size_t)B);
  for (int b = 0; b < B; ++b) {
    if (ids[b] < -1 || lens[b] < 0) return SPV_ERR_ARG;
    entries[E_WORDS * (size_t)b + E_GROUP] = -1;
    entries[E_WORDS * (size_t)b + E_RANK] = 0;
    if (ids[b] < 0 || lens[b] == 0) continue;
    const size_t g = index.emplace(std::make_pair(ids[b], lens[b]), groups.size()).first->second;
    if (g == groups.size()) groups.push_back({ids[b], lens[b], {}});
    entries[E_WORDS * (size_t)b + E_GROUP] = (int)g;
    entries[E_WORDS * (size_t)b + E_RANK] = (int)groups[g].members.size();
    groups[g].members.push_back(b);
  }
  std::vector<int32_t> gw, mw, sh, sw, tw;
  long long units = 0, maxp = 0, triples = 0;
  for (const Group& x : groups) {
    const long long tiles = ((long long)x.members.size() * G + kTile - 1) / kTile;
    if (triples + tiles * Hkv > 0x7fffffffLL / kTile) return SPV_ERR_UNSUPPORTED;
    const int32_t w[G_WORDS] = {x.sid, x.len, (int32_t)mw.size(), (int32_t)x.members.size(), (int32_t)tiles,
                                (int32_t)triples};
    gw.insert(gw.end(), w, w + G_WORDS);
    mw.insert(mw.end(), x.members.begin(), x.members.end());
    units += tiles * ((x.len + kUnit - 1) / kUnit);
    triples += tiles * Hkv;
    maxp = std::max<long long>(maxp, x.len);
  }
  tw.resize(T_WORDS * (size_t)triples);
  // Shares: equal runs of the units of all kv heads, groups and tiles (in that
  // order), two workgroups for each of the 256 CUs, or fewer where a share would be
  // shorter than two units.
  const long long total = units * Hkv;
  const long long nsh = total ? std::max(1LL, std::min(512LL, (total + 1) / 2) / 8) * 8 : 0;
  long long at = 0, share = 0;  // the unit in hand, and the share it belongs to
  auto first_unit = [&](long long s) { return s * total / nsh; };
  for (int h = 0; h < Hkv; ++h)
    for (size_t g = 0; g < groups.size(); ++g) {
      const long long n = (groups[g].len + kUnit - 1) / kUnit, tiles = gw[G_WORDS * g + G_NT];
      for (long long t = 0; t < tiles; ++t) {
        int32_t* const tile = &tw[T_WORDS * (size_t)(gw[G_WORDS * g + G_TILE0] + h * tiles + t)];
        tile[T_SEG] = (int32_t)(sw.size() / S_WORDS);
        for (long long u = 0; u < n;) {
          while (first_unit(share) <= at) {  // this unit opens share `share` (empty ones before it too)
            sh.push_back((int32_t)(sw.size() / S_WORDS));
            if (++share == nsh) break;
          }
          const long long end = share == nsh ? total : first_unit(share);
          const long long take = std::min(n - u, end - at);
          const int32_t w[S_WORDS] = {(int32_t)g, h, (int32_t)t, (int32_t)(u * kUnit),
                                      (int32_t)std::min<long long>((u + take) * kUnit, groups[g].len)};
          sw.insert(sw.end(), w, w + S_WORDS);
          u += take;
          at += take;
        }
        tile[T_COUNT] = (int32_t)(sw.size() / S_WORDS) - tile[T_SEG];
      }
    }
  while ((long long)sh.size() < nsh + 1) sh.push_back((int32_t)(sw.size() / S_WORDS));
  plan.assign(PH_WORDS, 0);
  plan[PH_MAGIC] = kPlanMagic;
  plan[PH_B] = B;
  plan[PH_C] = C;
  plan[PH_HQ] = Hq;
  plan[PH_HKV] = Hkv;
  plan[PH_BS] = bs;
  plan[PH_NG] = (int32_t)groups.size();
  plan[PH_NSH] = (int32_t)nsh;
  plan[PH_NSEG] = (int32_t)(sw.size() / S_WORDS);
  plan[PH_NT] = (int32_t)triples;
  plan[PH_MAXP] = (int32_t)maxp;
  auto add = [&](int word, const std::vector<int32_t>& v) {
    plan[word] = (int32_t)plan.size();
    plan.insert(plan.end(), v.begin(), v.end());
  };
  add(PH_GROUPS, gw);
  add(PH_MEMBERS, mw);
  add(PH_ENTRIES, entries);
  add(PH_SHARES, sh);
  add(PH_SEGS, sw);
  add(PH_TILES, tw);
  plan[PH_INTS] = (int32_t)plan.size();
  return SPV_OK;
}

// The entries' own ranges for contexts up to max_ctx.
void own_ranges(const int32_t* plan, int max_ctx, int* range, int* count) {
  const int bs = plan[PH_BS];
  int keys = std::max(256, (max_ctx + 31) / 32);
  keys = (keys + bs - 1) / bs * bs;
  *range = keys;
  *count = (max_ctx + keys - 1) / keys;
}

long long part_rows(const int32_t* plan, int max_ctx) {
  int range, count;
  own_ranges(plan, max_ctx, &range, &count);
  const long long G = (long long)plan[PH_C] * (plan[PH_HQ] / plan[PH_HKV]);
  return (long long)plan[PH_NSEG] * kTile + (long long)plan[PH_B] * plan[PH_HKV] * count * G;
}

// Floats of the (m, l) pairs at the workspace's head: whole 16-byte pieces, so that the rows behind them are aligned.
size_t ml_floats(size_t rows) { return (2 * rows + 3) / 4 * 4; }

template <int QT, int KT>
int launch_valu(const SharedParams& p, long long grid, hipStream_t s) {
  const size_t smem = valu_lds(p.d);
  if (smem > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(&shared_valu_kernel<QT, KT>),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != hipSuccess)
    return SPV_ERR_LAUNCH;
  hipLaunchKernelGGL((shared_valu_kernel<QT, KT>), dim3((unsigned)grid), dim3(kThreads), smem, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

template <int D, int KT>
int launch_mfma(const SharedParams& p, long long grid, hipStream_t s) {
  hipLaunchKernelGGL((shared_mfma_kernel<D, KT>), dim3((unsigned)grid), dim3(kThreads), 0, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

template <int QT, int LPR, bool VEC>
int launch_join(const SharedParams& p, hipStream_t s) {
  const long long rows = (long long)p.B * p.C * p.Hq, per = kThreads / LPR;
  hipLaunchKernelGGL((shared_join_kernel<QT, LPR, VEC>), dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads), 0, s,
                     p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

template <int QT>
int launch(const SharedParams& p, int kv_dtype, hipStream_t s) {
  const long long grid = p.shares + (long long)p.B * p.Hkv * p.own_tiles * p.own_max;
  int rc;
  // The matrix kernels apply the scale inside the exponent, to maxima of raw scores.
  const bool mfma = p.bs == 16 && (p.d == 64 || p.d == 128) && p.scale_log2 > 0.f && p.scale_log2 < INFINITY &&
                    ((QT == SPV_BF16 && (kv_dtype == SPV_BF16 || kv_dtype == SPV_FP8E4M3)) ||
                     (QT == SPV_F16 && kv_dtype == SPV_F16));
  if (mfma) {
    if constexpr (QT == SPV_BF16) {
      if (kv_dtype == SPV_BF16) rc = p.d == 64 ? launch_mfma<64, SPV_BF16>(p, grid, s) : launch_mfma<128, SPV_BF16>(p, grid, s);
      else rc = p.d == 64 ? launch_mfma<64, SPV_FP8E4M3>(p, grid, s) : launch_mfma<128, SPV_FP8E4M3>(p, grid, s);
    } else if constexpr (QT == SPV_F16) {
      rc = p.d == 64 ? launch_mfma<64, SPV_F16>(p, grid, s) : launch_mfma<128, SPV_F16>(p, grid, s);
    }
  } else switch (kv_dtype) {
    case SPV_F32: rc = launch_valu<QT, SPV_F32>(p, grid, s); break;
    case SPV_BF16: rc = launch_valu<QT, SPV_BF16>(p, grid, s); break;
    case SPV_F16: rc = launch_valu<QT, SPV_F16>(p, grid, s); break;
    default: rc = launch_valu<QT, SPV_FP8E4M3>(p, grid, s); break;
  }
  if (rc != SPV_OK) return rc;
  if (p.d == 128) return launch_join<QT, 32, true>(p, s);
  if (p.d == 64) return launch_join<QT, 16, true>(p, s);
  return launch_join<QT, 64, false>(p, s);
}

}  // namespace

extern "C" {

int64_t spv_shared_attn_plan(const int32_t* prefix_ids, const int32_t* prefix_lens, int32_t B, int32_t C,
                             int32_t num_q_heads, int32_t num_kv_heads, int32_t block_size, int32_t* plan,
                             int64_t plan_ints) {
  if (!prefix_ids || !prefix_lens || B < 1 || B > 65535 || C < 1 || num_kv_heads < 1 ||
      num_q_heads < num_kv_heads || num_q_heads % num_kv_heads || block_size < 1 ||
      (long long)C * num_q_heads > (1 << 20) || (long long)B * C * num_q_heads > (1LL << 30))
    return SPV_ERR_ARG;
  try {
    std::vector<int32_t> p;
    const int rc = make_plan(p, prefix_ids, prefix_lens, B, C, num_q_heads, num_kv_heads, block_size);
    if (rc != SPV_OK) return rc;
    if (!plan) return (int64_t)p.size();
    if (plan_ints < (int64_t)p.size()) return SPV_ERR_WORKSPACE;
    for (size_t i = 0; i < p.size(); ++i) plan[i] = p[i];
    return (int64_t)p.size();
  } catch (...) {  // no memory on the host
    return SPV_ERR_UNSUPPORTED;
  }
}

size_t spv_shared_attn_workspace_bytes(const int32_t* plan_host, int32_t head_dim, int32_t max_ctx) {
  if (!plan_host || plan_host[PH_MAGIC] != kPlanMagic || head_dim < 1 || max_ctx < plan_host[PH_C]) return 0;
  const size_t rows = (size_t)part_rows(plan_host, max_ctx);
  return (ml_floats(rows) + rows * head_dim) * sizeof(float);
}

int spv_shared_attn(void* out, const void* q, int q_dtype, const void* k_pool, const void* v_pool, int kv_dtype,
                    const float* kv_scales, const int32_t* block_tables, int32_t max_blocks_per_seq,
                    const int32_t* seq_ids, const int32_t* start_pos, const int32_t* seq_lens, int32_t* ctr,
                    int32_t B, int32_t C, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                    int32_t block_size, int32_t layer, int32_t capacity, int32_t max_ctx, float scale,
                    const int32_t* plan_host, const int32_t* plan, void* workspace, size_t workspace_bytes,
                    void* stream) {
  if (!out || !q || !k_pool || !v_pool || !block_tables || !seq_ids || !start_pos || !plan_host || !plan ||
      !workspace)
    return SPV_ERR_ARG;
  if (q_dtype != SPV_F32 && q_dtype != SPV_BF16 && q_dtype != SPV_F16) return SPV_ERR_ARG;
  if (dtype_size(kv_dtype) == 0 || (kv_dtype == SPV_FP8E4M3 && !kv_scales)) return SPV_ERR_ARG;
  const int32_t* h = plan_host;
  if (h[PH_MAGIC] != kPlanMagic || h[PH_B] != B || h[PH_C] != C || h[PH_HQ] != num_q_heads ||
      h[PH_HKV] != num_kv_heads || h[PH_BS] != block_size)
    return SPV_ERR_ARG;
  if (head_dim < 1 || head_dim > 256 || layer < 0 || capacity < 1 || max_ctx < C || max_ctx > (1 << 30)) return SPV_ERR_ARG;
  const int longest = std::max(max_ctx, h[PH_MAXP]);
  if (max_blocks_per_seq < (longest + block_size - 1) / block_size) return SPV_ERR_ARG;
  if (workspace_bytes < spv_shared_attn_workspace_bytes(h, head_dim, max_ctx)) return SPV_ERR_WORKSPACE;
  SharedParams p{};
  p.out = out;
  p.q = q;
  p.kpool = k_pool;
  p.vpool = v_pool;
  p.scales = kv_scales;
  p.tables = block_tables;
  p.seq_ids = seq_ids;
  p.start = start_pos;
  p.lens = seq_lens;
  p.ctr = ctr;
  p.plan = plan;
  p.maxb = max_blocks_per_seq;
  p.B = B;
  p.C = C;
  p.Hq = num_q_heads;
  p.Hkv = num_kv_heads;
  p.ratio = num_q_heads / num_kv_heads;
  p.G = C * p.ratio;
  p.d = head_dim;
  p.bs = block_size;
  p.layer = layer;
  p.cap = capacity;
  p.shares = h[PH_NSH];
  p.max_ctx = max_ctx;
  own_ranges(h, max_ctx, &p.own_range, &p.own_max);
  p.own_tiles = (p.G + kTile - 1) / kTile;
  p.own_part = (long long)h[PH_NSEG] * kTile;
  const long long rows = part_rows(h, max_ctx);
  // both grids: at most 2^32 threads
  if (p.shares + (long long)B * num_kv_heads * p.own_tiles * p.own_max > (1LL << 23) ||
      (long long)B * C * num_q_heads > (1LL << 23))
    return SPV_ERR_UNSUPPORTED;
  p.part_ml = static_cast<float*>(workspace);
  p.part_o = p.part_ml + ml_floats((size_t)rows);
  p.scale_log2 = scale * kLog2e;
  hipStream_t s = (hipStream_t)stream;
  if (q_dtype == SPV_F32) return launch<SPV_F32>(p, kv_dtype, s);
  if (q_dtype == SPV_BF16) return launch<SPV_BF16>(p, kv_dtype, s);
  return launch<SPV_F16>(p, kv_dtype, s);
}

}  // extern "C"
