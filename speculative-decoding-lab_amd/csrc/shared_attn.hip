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
// 256, a prefix's keys into equal ranges; a segment is one tile over one range,
// walked by one workgroup, and leaves a partial. Further workgroups walk the
// entries' own keys, one per (entry, kv head, 64 of its rows, range). A second
// launch joins each row's partials. The segments are listed on the host (the
// prefixes and their lengths change when a request is admitted, not between
// rounds); the entries' own lengths are read on the device.
//
// Matrix path (bf16 queries over bf16 or fp8 pages, fp16 over fp16, fp32 over fp32,
// head_dim 64 or 128, 16-token blocks, a finite positive scale). Own keys, segments of
// at most 64 rows and all of fp32 take pages straight into operand registers, the waves
// sharing them out. Larger segments: a workgroup of eight waves
// takes a tile, 32 rows per wave, and stages 64 keys at a time in LDS, so that a
// key read from the L2 once serves 256 rows. Per 16-key page and 16 rows
//   S^T = K Q^T    v_mfma_f32_16x16x32, A = 16 keys x 32 dims, B = Q^T fragments
//                  that stay in registers for the whole segment;
//   O^T += V^T P^T v_mfma_f32_16x16x32_f16 over two pages, P in fp16.
// S^T's accumulator layout is P^T's operand layout (lane l: keys 4 (l / 16) .. + 3
// of row l % 16), so the softmax moves no data between lanes. P in bf16 (8 bits)
// would miss the library's bf16 bar (2e-3 per sequence, of which rounding the
// output alone takes 1.7e-3); fp16 has 11 bits. (fp16 outputs, whose rounding takes 2.1e-4, are
// 2.85e-4 off float64 so; in two halves P would add nothing to 2.1e-4, and 7168 x 2 rows over 8192
// keys would take 137 us for 114, 1008 x 2 of head_dim 64 over 32768 keys 49 for 41.)
// bf16 values are staged as fp16 times a power of two per segment, chosen from the first tile's largest |v|
// (which lands in [2^8, 2^9): every value from 2^-25 of it up is exact, a smaller
// one is off by at most 2^-33 of it). Where a later value would pass fp16's range, a page has 32
// dims that all lie below 2^-12 of that largest (a row whose weight is there would lose bits), or the
// first tile is all zeros, the segment is walked again page by page as own keys are, in any
// range (7168 x 2 rows over 8192 keys 280 us where every segment is, 114 where none). fp16 values
// are staged as they are: beside values of 2^15 P's 2^-32 is 2^-17, in either walk. fp8 codes are
// fp16 values; a block's K scale goes into the exponent's multiplier, its V scale, over
// the segment's largest, as a logarithm into the addend, so that P carries it; segments whose V scales
// (zeros aside) lie more than 2^12 apart are walked page by page, too (P in two halves of bf16, with
// fp32's exponents).
//
// What bounds it: with long prefixes and many rows the walk (7168 x 2 bf16 rows: each further
// 8192 keys take 49 us, 1.2 PFLOP/s; 6272 x 2 of head_dim 64 0.73, over fp8 0.76 to 0.79) and
// its segments' starts and ends: 7168 x 2 rows over 8192 keys and up to 1024 own keys an entry (64
// GFLOP) take 104 us and 9 in the join. With short ones the
// launches, the first pages' round trips and the partials, which are written and
// read at the rate of memory: 1152 x 2 rows over 2048 keys 21 us and 5 in the join.
#include <math.h>

#include <algorithm>
#include <map>
#include <utility>
#include <vector>

#include "spv_common.h"

using namespace spv;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The plan: a header, then the segments -- ordered by group, kv head, range, tile, so
// that neighbours read the same keys --, the members of the groups (batch
// entries), and each entry's place.
enum : int {
  PH_MAGIC = 0,
  PH_INTS,  // length of the plan
  PH_B,
  PH_C,
  PH_HQ,
  PH_HKV,
  PH_BS,
  PH_NSEG,  // segments
  PH_MAXP,  // longest prefix
  PH_SEGS,
  PH_MEMBERS,
  PH_ENTRIES,
  PH_OWN,   // keys of an own range at least
  PH_TILE,  // rows of a tile
  PH_WORDS
};
constexpr int kPlanMagic = 0x53505235;
// A segment: sequence and length of the prefix, kv head, first member, first row of
// the tile and its rows, the keys.
enum : int { S_SID = 0, S_LEN, S_HEAD, S_FIRST, S_ROW0, S_ROWS, S_KEY0, S_KEY1, S_WORDS };
// An entry: the group's first segment (-1: no prefix), its tiles, ranges, the entry's rank in it.
enum : int { E_SEG = 0, E_TILES, E_RANGES, E_RANK, E_WORDS };
constexpr int kTile = 256;    // rows of a prefix tile (fp32: 64, 128 or 256)
constexpr int kUnit = 64;     // keys
constexpr int kOwnRows = 64;  // rows of an entry that a workgroup takes over its own keys
constexpr int kPagesRows = 64;  // segments of at most so many rows are walked like own keys

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
  const int32_t* segs;  // the plan's sections
  const int32_t* members;
  const int32_t* entries;
  float* part_o;   // partial rows x d
  float* part_ml;  // partial rows x 2
  int maxb, B, C, Hq, Hkv, ratio, G, d, bs, layer, cap;
  int tile;                // rows of a segment
  int nseg, seg_wgs;       // segments, and their workgroups (a multiple of 8)
  int own_range, own_max;  // keys per own range (whole blocks), ranges per entry at most
  int own_tiles;           // tiles of an entry's rows
  int max_ctx;
  long long own_part;      // first partial row of the own ranges
  float scale_log2;
};

// One piece of work: rows [row0, row0 + rows) of a group's (or one entry's) row
// order over keys [key0, key1) of one sequence.
struct Item {
  int first;  // the group's first member, or -1: an entry's own keys
  int sid, b, h, row0, rows, key0, key1;
  int start;       // own keys: row j sees keys <= start + j
  long long part;  // its first partial row
};

__device__ __forceinline__ void flag_bad_read(const SharedParams& p, int b) {
  if (p.ctr) p.ctr[CTR_BAD_READ] = b + 1;
}

// The segment of workgroup `id`: workgroups go round-robin over the 8 XCDs, each of
// which takes an eighth of the segments in a row, so that its L2 serves one range
// of keys to workgroups that walk it side by side. False past the last one.
__device__ __forceinline__ bool segment_item(const SharedParams& p, int id, Item& it) {
  const int seg = (id & 7) * (p.seg_wgs >> 3) + (id >> 3);
  if (seg >= p.nseg) return false;
  const int32_t* s = p.segs + (size_t)seg * S_WORDS;
  it.first = s[S_FIRST];
  it.sid = s[S_SID];
  it.h = s[S_HEAD];
  it.row0 = s[S_ROW0];
  it.rows = s[S_ROWS];
  it.key0 = s[S_KEY0];
  it.key1 = s[S_KEY1];
  it.start = 0x3fffffff;
  it.b = p.members[it.first];
  it.part = (long long)seg * p.tile;
  if (threadIdx.x == 0 && p.lens && p.lens[it.sid] < s[S_LEN]) flag_bad_read(p, it.b);
  return true;
}

// Own work `o`: false where the range has no keys.
__device__ __forceinline__ bool own_item(const SharedParams& p, int o, Item& it) {
  const int s = o % p.own_max, bht = o / p.own_max, t = bht % p.own_tiles, bh = bht / p.own_tiles;
  it.first = -1;
  it.b = bh / p.Hkv;
  it.h = bh - it.b * p.Hkv;
  it.sid = p.seq_ids[it.b];
  it.start = p.start[it.b];
  const int L = it.start + p.C, seen = min(max(L, 0), p.max_ctx);
  if (threadIdx.x == 0 && s == 0 && it.h == 0 && (it.start < 0 || L > p.max_ctx || (p.lens && p.lens[it.sid] < L)))
    flag_bad_read(p, it.b);
  it.row0 = t * kOwnRows;
  it.rows = min(kOwnRows, p.G - it.row0);
  it.key0 = s * p.own_range;
  it.key1 = min(it.key0 + p.own_range, seen);
  it.part = p.own_part + ((long long)bh * p.own_max + s) * p.G + it.row0;
  return it.key0 < it.key1;
}

// Row R of an item's row order: its entry, chunk token and q head.
__device__ __forceinline__ void row_at(const SharedParams& p, const Item& it, int R, int& b, int& j, int& hq) {
  const int m = it.first >= 0 ? R / p.G : 0, r = R - m * p.G;
  const int member = p.members[max(it.first, 0) + m];  // (the entries' section follows the members')
  b = it.first >= 0 ? member : it.b;
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

// MD: a bound on head_dim; TH: threads of the workgroup (at least 256).
template <int QT, int KT, int MD, int TH>
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
    for (int i = threadIdx.x; i < nr * d; i += TH) {
      const int rr = i / d, e = i - rr * d;
      int b, j, hq;
      row_at(p, it, it.row0 + r0 + rr, b, j, hq);
      Qs[rr * pitch + e] = load_elem<QT>(p.q, (((size_t)b * p.C + j) * p.Hq + hq) * d + e) * p.scale_log2;
      if (e == 0) Lim[rr] = it.first >= 0 ? it.start : it.start + j;
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
      for (int i = threadIdx.x; i < nt * d; i += TH) {
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
      for (int i = threadIdx.x; i < nr * kKeys; i += TH) {
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

// Workgroups [0, seg_wgs) walk prefixes, the others entries' own keys: those are short
// and fill the CUs that the prefixes leave.
template <int QT, int KT>
__global__ __launch_bounds__(kThreads) void shared_valu_kernel(SharedParams p) {
  extern __shared__ float smem[];
  const int id = blockIdx.x;
  Item it;
  if (id < p.seg_wgs ? segment_item(p, id, it) : own_item(p, id - p.seg_wgs, it))
    valu_item<QT, KT, kMaxD, kThreads>(p, it, smem);
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
// its sums are rescaled: P stays below 2^8.
constexpr float kSlack = 8.f;
// Where P goes in fp16, the reference lies this much below the maximum that it was taken from: P
// is at most 2^15 then, has fp16's whole 11 bits from 2^-21 of the maximum's up, and is off by at
// most 2^-32 of that below.
constexpr float kShift = 7.f;
// The tiled walk over fp8 pages takes V scales down to this fraction of a segment's largest. It puts
// the ratio into P: at 2^-12 a row whose weight is on such a page still has P of 2^-5, and what P
// loses on other pages' small weights, 2^-32 times their values, is 2^-20 of its own.
constexpr float kScaleRange = 0x1p-12f;

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
// The staging power for a largest finite |v| of mx > 0: mx 2^k in [2^8, 2^9).
__device__ __forceinline__ int stage_exponent(float mx) {
  int e;
  frexpf(mx, &e);
  return min(126, max(-126, 9 - e));
}

#define SPV_INLINE __attribute__((always_inline))  // on the walks' lambdas: their operands stay in registers
constexpr int kWaves = 8;
constexpr int kMfmaThreads = 64 * kWaves;

template <int D>
struct Lds {
  // 32 bytes of padding on a K row and a V^T row: their 16-byte reads meet no bank twice.
  static constexpr int KP = D + 16, VP = kUnit + 16;
  static constexpr int kK = kUnit * KP, kV = D * VP;  // elements of a slot
  static constexpr size_t kWalk = 2 * (size_t)(2 * kK + 3 * kV);
  static constexpr int kJP = D / 2 + 4;  // own keys: half of a wave's row of sums, padded
  static constexpr size_t kJoinRows = kWaves * 32 * (size_t)kJP * 4, kJoin = kJoinRows + kWaves * 32 * 8;
  static constexpr size_t kBytes = (kWalk > kJoin ? kWalk : kJoin) + 4 * kWaves;
};

// What both walks know of the call and the lane.
template <int D, int KT>
struct Walk {
  static constexpr bool kF16 = KT == SPV_F16, kFp8 = KT == SPV_FP8E4M3, kF32 = KT == SPV_F32;
  static constexpr int QT = kF16 ? SPV_F16 : kF32 ? SPV_F32 : SPV_BF16;
  static constexpr int ES = kFp8 ? 1 : kF32 ? 4 : 2;
  static constexpr int KS = kF32 ? D / 16 : D / 32, MT = D / 16, NT = 2;  // KS: 16-byte pieces of a row per lane
  const SharedParams& p;
  uint8_t* const smem;
  uint32_t* const sMax;
  const int tid, lane, w, i16, g;
  const float sl2, inv_sl2;

  __device__ __forceinline__ Walk(const SharedParams& p_, uint8_t* smem_, int tid_)
      : p(p_), smem(smem_), sMax(reinterpret_cast<uint32_t*>(smem_ + Lds<D>::kBytes) - kWaves), tid(tid_),
        lane(tid_ & 63), w(__builtin_amdgcn_readfirstlane(tid_ >> 6)), i16(tid_ & 15), g((tid_ & 63) >> 4),
        sl2(p_.scale_log2), inv_sl2(1.f / p_.scale_log2) {}

  // The query fragments of the lane's rows r0 + 16 nt + i16 of an item: B operands, 8
  // dims from 32 ks + 8 g on (fp32: 4 dims from 16 ks + 4 g on).
  __device__ __forceinline__ void load_q(const Item& it, int r0, uint4 (&qf)[NT][KS], int (&lim)[NT], bool (&valid)[NT]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int R = r0 + nt * 16 + i16;
      valid[nt] = R < it.rows;
      int b, j, hq;
      row_at(p, it, it.row0 + min(R, it.rows - 1), b, j, hq);
      lim[nt] = it.first >= 0 ? it.start : it.start + j;
      const uint8_t* q =
          static_cast<const uint8_t*>(p.q) + (((size_t)b * p.C + j) * p.Hq + hq) * (D * (kF32 ? 4 : 2)) + 16 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[nt][ks] = *reinterpret_cast<const uint4*>(q + 64 * ks);
    }
  }
  __device__ __forceinline__ f32x4_t mfma_qk(uint4 k, uint4 q, f32x4_t c) const {
    if constexpr (kF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k), __builtin_bit_cast(f16x8_t, q), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q), c, 0, 0, 0);
  }
  __device__ __forceinline__ int safe_id(const Item& it, int phys) const {
    if ((unsigned)phys < (unsigned)p.cap) return phys;
    flag_bad_read(p, it.b);
    return 0;
  }
  __device__ __forceinline__ float2 scales_of(int phys) const {
    return *reinterpret_cast<const float2*>(p.scales + ((size_t)p.layer * p.cap + phys) * 2);
  }
  // A block's page of kv head h, counted in pages (the host checks that they fit 31 bits), and its address.
  __device__ __forceinline__ int page_of(int phys, int h) const { return (p.layer * p.cap + phys) * p.Hkv + h; }
  __device__ __forceinline__ const uint8_t* page(const void* pool, int index) const {
    return static_cast<const uint8_t*>(pool) + (size_t)(uint32_t)index * (16 * D * ES);
  }
  // The workgroup's largest of either half of m (16 bits each), in every thread.
  __device__ __forceinline__ uint32_t wg_max2(uint32_t m) {
    const auto larger = [](uint32_t a, uint32_t b) {
      return __builtin_bit_cast(uint32_t,
                                __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
    };
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = larger(m, (uint32_t)__shfl_xor((int)m, o, 64));
    __syncthreads();
    if (lane == 0) sMax[w] = m;
    __syncthreads();
    m = sMax[0];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) m = larger(m, sMax[k]);
    return m;
  }

  // ---- a segment of a prefix: 256 rows, 32 per wave, 64 keys at a time in LDS. False
  // where bf16 values do not fit the staging (above), the V scales of fp8 pages lie too far apart, or
  // an fp16 value that makes a sum so is not finite: nothing is written then.
  __device__ __forceinline__ bool prefix(const Item& it) {
    using LD = Lds<D>;
    constexpr int KP = LD::KP, VP = LD::VP;
    uint16_t* const sK = reinterpret_cast<uint16_t*>(smem);
    uint16_t* const sV = sK + 2 * LD::kK;
    const f16x2_t ones = f16x2_t{(_Float16)1.f, (_Float16)1.f};
    // Wave groups: waves 0-3 and 4-7, one of each per SIMD.
    const int grp = w >> 2, gt = tid & 255, gw = w & 3;
    const int h = __builtin_amdgcn_readfirstlane(it.h), key0 = __builtin_amdgcn_readfirstlane(it.key0),
              key1 = __builtin_amdgcn_readfirstlane(it.key1);
    const int pages = (key1 - key0 + 15) >> 4, n = (key1 - key0 + kUnit - 1) / kUnit;
    const int32_t* table = p.tables + (size_t)__builtin_amdgcn_readfirstlane(it.sid) * p.maxb + (key0 >> 4);

    // Page numbers (and an fp8 page's scales) of 64 pages, 16 tiles, in the lanes of a
    // register, the next 64 ids read with every tile (a branch around the read costs
    // more than the read); pages past the range repeat its last one.
    int ids = 0, idn = 0;
    float ksc = 1.f, vsc = 1.f, vref = 1.f;  // vref, fp8: a bound on the range's V scales
    auto read_ids = [&](int first) SPV_INLINE { return table[min(first + lane, pages - 1)]; };
    auto open_window = [&](int raw) SPV_INLINE {
      const int phys = safe_id(it, raw);
      ids = page_of(phys, h);
      if constexpr (kFp8) {
        const float2 s = scales_of(phys);
        ksc = s.x;
        vsc = s.y;
      }
    };
    int raw = read_ids(0);
    uint4 qf[NT][KS];
    int lim[NT];
    bool valid[NT];
    load_q(it, w * 32, qf, lim, valid);

    // Staging: each group stages half of a tile. K: 16-byte pieces of a page in
    // memory order. V: (dim, page pair, half) items: 8 keys of the even and 8 of the
    // odd page. In a V^T row key 4 gg + j of page 2 q + hh sits at 32 q + 8 gg +
    // 4 hh + j, so that lane group gg's 16-byte read holds its keys of both pages.
    constexpr int kKP = kUnit * D * ES / 16, kKN = kKP / 2 / 256;  // K pieces of a tile, per thread
    constexpr int kVI = 4 * D, kVN = (kVI / 2 + 255) / 256;        // V items of a tile, per thread
    static_assert(kKP / 2 % 256 == 0 || kKP / 2 < 256, "whole pieces per thread");
    constexpr int kKN1 = kKN ? kKN : 1;
    struct Stage {
      u32x4_t k[kKN1];
      u32x4_t v[kVN][2];  // fp8: the first 8 bytes
    };
    constexpr int kPer = D * ES;  // 16-byte pieces of a page
    // Group threads beyond a half's pieces (the smallest tiles) repeat one of them.
    auto k_piece = [&](int i) SPV_INLINE { return grp * (kKP / 2) + (gt + i * 256) % (kKP / 2); };
    auto v_item = [&](int i) SPV_INLINE { return grp * (kVI / 2) + (gt + i * 256) % (kVI / 2); };
    auto k_page = [&](int i) SPV_INLINE { return (grp * (kKP / 2) + (gw * 64 + i * 256) % (kKP / 2)) / kPer; };  // of the wave's pieces
    auto v_pair = [&](int i) SPV_INLINE { return (grp * (kVI / 2) + (gw * 64 + i * 256) % (kVI / 2)) / (2 * D); };
    auto load = [&](Stage& S, int t) SPV_INLINE {
#pragma unroll
      for (int i = 0; i < kKN1; ++i) {
        const int pg = __builtin_amdgcn_readlane(ids, (4 * t + k_page(i)) & 63);
        S.k[i] = *reinterpret_cast<const u32x4_t*>(page(p.kpool, pg) + 16 * (k_piece(i) % kPer));
      }
#pragma unroll
      for (int i = 0; i < kVN; ++i) {
        const int q = v_pair(i), c = v_item(i) % (2 * D);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int pg = __builtin_amdgcn_readlane(ids, (4 * t + 2 * q + hh) & 63);
          const uint8_t* v = page(p.vpool, pg) + 8 * ES * c;
          if constexpr (kFp8) {
            const uint2 x = *reinterpret_cast<const uint2*>(v);
            S.v[i][hh] = u32x4_t{x.x, x.y, 0u, 0u};
          } else {
            S.v[i][hh] = *reinterpret_cast<const u32x4_t*>(v);
          }
        }
      }
    };
    // The window of tile t, before its loads (tiles are loaded in order).
    auto window = [&](int t) SPV_INLINE {
      if (t < n && (t & 15) == 0) open_window(idn);
      idn = read_ids(4 * ((t & ~15) + 16));
    };
    auto load_next = [&](Stage& S, int t) SPV_INLINE {
      window(t);
      load(S, min(t, n - 1));
    };
    float vs = 1.f;  // bf16: the staging factor 2^vk
    int vk = 0;
    // bf16, as bits of |v|: a little less than what a page's largest has to reach, what none may
    // pass, the largest so far (of either half of a word), and whether one of the wave's pages (32
    // dims of it) is too small.
    uint32_t low2 = 0, top = 0, vmax = 0, small = 0;
    // Zeroes the values of keys past the range's end.
    auto edge = [&](Stage& S, int t) SPV_INLINE {
      const int t0 = key0 + t * kUnit;
      if (t0 + kUnit <= key1) return;
#pragma unroll
      for (int i = 0; i < kVN; ++i) {
        const int q = v_pair(i), half = gt & 1;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          u32x4_t x = S.v[i][hh];
          const int k0 = t0 + 32 * q + 16 * hh + 8 * half;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            constexpr uint32_t kMask = kFp8 ? 0xffu : 0xffffu;
            x[e * ES / 4] &= k0 + e >= key1 ? ~(kMask << (8 * (e * ES % 4))) : ~0u;
          }
          S.v[i][hh] = x;
        }
      }
    };
    // bf16 values to fp16, in place, in the softmax's phase: beside the matrix
    // instructions they left no registers for the operands' read-ahead (0.69 PFLOP/s).
    // A wave's 64 pieces are 32 dims of a page.
    auto convert = [&](Stage& S) SPV_INLINE {
      if constexpr (!kF16 && !kFp8) {
#pragma unroll
        for (int i = 0; i < kVN; ++i)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            u32x4_t x = S.v[i][hh];
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t y = x[e];
              most = max_abs2(y, most);
              x[e] = pack2_f16(__uint_as_float(y << 16) * vs, __uint_as_float(y & 0xffff0000u) * vs);
            }
            S.v[i][hh] = x;
            vmax = max_abs2(most, vmax);
            const u16x2_t over = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2_t, most),
                                                               __builtin_bit_cast(u16x2_t, low2));
            small |= (uint32_t)(__ballot(most != 0) != 0) & (uint32_t)(__ballot(__builtin_bit_cast(uint32_t, over) != 0) == 0);
          }
      }
    };
    auto store = [&](Stage& S, int kslot, int vslot) SPV_INLINE {
      uint16_t* const K = sK + kslot * LD::kK;
      uint16_t* const V = sV + vslot * LD::kV;
#pragma unroll
      for (int i = 0; i < kKN1; ++i) {
        const int pi = k_page(i), c = k_piece(i) % kPer;
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
        const int q = v_pair(i), c = v_item(i) % (2 * D), dim = c >> 1, half = c & 1;
        uint2 y[2][2];  // [page][keys 0-3, 4-7 of the half]
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const u32x4_t x = S.v[i][hh];
          uint32_t z[4];
          if constexpr (kF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = x[e];
          } else if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              z[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[e], 1.f, false));
              z[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[e], 1.f, true));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = x[e];
          }
          y[hh][0] = make_uint2(z[0], z[1]);
          y[hh][1] = make_uint2(z[2], z[3]);
        }
        uint16_t* const row = &V[dim * VP + 32 * q + 16 * half];
        *reinterpret_cast<uint4*>(row) = make_uint4(y[0][0].x, y[0][0].y, y[1][0].x, y[1][0].y);
        *reinterpret_cast<uint4*>(row + 8) = make_uint4(y[0][1].x, y[0][1].y, y[1][1].x, y[1][1].y);
      }
    };

    f32x4_t o[MT][NT];
    float m[NT], l[NT], thr[NT];  // thr: the score above which m must grow
    f32x4_t sc[4][NT];            // S^T of the tile in the walk
    uint32_t ph[2][NT][4];        // its P, two pages an operand
    // fp8, of the window of the tile in the walk: a page's K scale times the softmax's, log2 of
    // its V scale over vref, and the inverse of that ratio. Pages of scale 0, of zeros, count as
    // 2^-100.
    float ks_t = 1.f, vl_t = 0.f, vi_t = 1.f;
    auto pv = [&](int vslot) SPV_INLINE {
      const uint16_t* V = sV + vslot * LD::kV;
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const f16x8_t va =
              __builtin_bit_cast(f16x8_t, *reinterpret_cast<const uint4*>(&V[(16 * mt + i16) * VP + 32 * q + 8 * g]));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            o[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                va, __builtin_bit_cast(f16x8_t, make_uint4(ph[q][nt][0], ph[q][nt][1], ph[q][nt][2], ph[q][nt][3])),
                o[mt][nt], 0, 0, 0);
        }
    };
    auto qk = [&](int kslot) SPV_INLINE {
      const uint16_t* K = sK + kslot * LD::kK;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[kt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const uint4 kf = *reinterpret_cast<const uint4*>(&K[(16 * kt + i16) * KP + 32 * ks + 8 * g]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[kt][nt] = mfma_qk(kf, qf[nt][ks], sc[kt][nt]);
        }
      }
    };
    auto softmax = [&](int t) SPV_INLINE {
      // fp8: scores stay raw codes' products; a page's K scale goes into the exponent's
      // multiplier and its V scale, as a logarithm, into the addend.
      float slf[4], lv[4], vi[4];
      if constexpr (kFp8) {
        if ((t & 15) == 0) {
          ks_t = ksc * sl2;
          if (ks_t == 0.f) ks_t = 1e-38f;  // (a masked -inf times 0 would be NaN)
          const float ratio = vref > 0.f ? vsc / vref : 0.f;
          vl_t = ratio == 0.f ? -100.f : __builtin_amdgcn_logf(ratio);
          vi_t = __builtin_amdgcn_exp2f(-vl_t);
        }
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const int at = (4 * t + kt) & 63;
          slf[kt] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_t), at));
          lv[kt] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vl_t), at));
          vi[kt] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vi_t), at));
        }
      }
      const int t0 = key0 + t * kUnit;
      if (t0 + kUnit > key1) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
              if (t0 + 16 * kt + 4 * g + jj >= key1) sc[kt][nt][jj] = -INFINITY;
      }
      float mx[NT];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (kFp8) {  // in log2 units
          float a[4];
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
            a[kt] = slf[kt] * max3_raw(max3_raw(sc[kt][nt][0], sc[kt][nt][1], sc[kt][nt][2]), sc[kt][nt][3],
                                       sc[kt][nt][3]);
          mx[nt] = max3_raw(max3_raw(a[0], a[1], a[2]), a[3], a[3]);
        } else {
          float a0 = max3_raw(sc[0][nt][0], sc[0][nt][1], sc[0][nt][2]);
          float a1 = max3_raw(sc[0][nt][3], sc[1][nt][0], sc[1][nt][1]);
          float a2 = max3_raw(sc[1][nt][2], sc[1][nt][3], sc[2][nt][0]);
          float a3 = max3_raw(sc[2][nt][1], sc[2][nt][2], sc[2][nt][3]);
          float a4 = max3_raw(sc[3][nt][0], sc[3][nt][1], sc[3][nt][2]);
          a0 = max3_raw(a0, a1, a2);
          a3 = max3_raw(a3, a4, sc[3][nt][3]);
          mx[nt] = fmaxf(a0, a3);
        }
        grow |= mx[nt] > thr[nt];
      }
      if (__any(grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float a = fmaxf(mx[nt], __shfl_xor(mx[nt], 16, 64));
          a = fmaxf(a, __shfl_xor(a, 32, 64));
          const float m_new = fmaxf(m[nt], (kFp8 ? a : a * sl2) - kShift);
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nt] - m_new);
          l[nt] *= alpha;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) o[mt][nt] *= alpha;
          m[nt] = m_new;
          thr[nt] = kFp8 ? m_new + (kShift + kSlack) : (m_new + (kShift + kSlack)) * inv_sl2;
        }
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float mu = m[nt] == -INFINITY ? 0.f : m[nt];
          const float mul = kFp8 ? slf[kt] : sl2, add = kFp8 ? lv[kt] - mu : -mu;
          float e[4];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) e[jj] = __builtin_amdgcn_exp2f(fmaf(sc[kt][nt][jj], mul, add));
          if constexpr (kFp8) l[nt] = fmaf((e[0] + e[1]) + (e[2] + e[3]), vi[kt], l[nt]);
          const uint32_t p01 = pack2_f16(e[0], e[1]), p23 = pack2_f16(e[2], e[3]);
          ph[kt >> 1][nt][2 * (kt & 1)] = p01;
          ph[kt >> 1][nt][2 * (kt & 1) + 1] = p23;
          if constexpr (!kFp8) {  // the sum takes P as it enters P V
            l[nt] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p01), ones, l[nt], false);
            l[nt] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p23), ones, l[nt], false);
          }
        }
      }
    };
    // A phase ends at a workgroup barrier that no instruction is scheduled across.
    auto phase_end = []() SPV_INLINE {
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
    };
    // The walk. Group 0 runs phases M(0), V(0), M(1), V(1), ... and group 1 the same
    // one phase later, a barrier after each, so that on every SIMD one wave's
    // softmax runs beside the other's matrix instructions:
    //   M(t): stage the group's half of tile t + 1, load that of tile t + 3;
    //         O^T += V^T P^T of tile t - 1, then S^T of tile t
    //   V(t): softmax of tile t
    // The staging goes with the matrix instructions, which leave the other issue ports
    // free (beside the softmax, the longer phase, it took a third more time). Tile x
    // is staged in M(x - 1), its K read in M(x) and its V in M(x + 1) of either group:
    // two K slots, three V slots.
    Stage st0, st1;
    {
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
      idn = raw;
      load_next(st0, 0);
      load_next(st1, 1);
      if constexpr (kFp8) {
        float mx = 0.f, mn = INFINITY;  // of scales that are not 0 (pages of zeros)
        for (int pg = tid; pg < pages; pg += kMfmaThreads) {
          const int phys = table[pg];
          if ((unsigned)phys >= (unsigned)p.cap) continue;
          const float s = scales_of(phys).y;
          mx = fmaxf(mx, s);
          if (s > 0.f) mn = fminf(mn, s);
        }
        // both over the workgroup at once, as bf16: the largest rounded up, the smallest down
        const uint32_t both =
            wg_max2((__float_as_uint(mx) + 0xffffu) >> 16 | (0xffffu - (__float_as_uint(mn) >> 16)) << 16);
        vref = __uint_as_float(both << 16);
        if (__uint_as_float((0xffffu - (both >> 16)) << 16) < vref * kScaleRange) return false;
      }
      if constexpr (!kF16 && !kFp8) {
        uint32_t mx = 0;  // the largest finite |v| of the first tile
        edge(st0, 0);
#pragma unroll
        for (int i = 0; i < kVN; ++i)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const u32x4_t x = st0.v[i][hh];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t lo = x[e] & 0x7fffu, hi = (x[e] >> 16) & 0x7fffu;
              mx = max(mx, lo < 0x7f80u ? lo : 0u);
              mx = max(mx, hi < 0x7f80u ? hi : 0u);
            }
          }
        mx = __builtin_amdgcn_readfirstlane(wg_max2(mx));
        if (mx == 0) return false;  // all zero: nothing to choose the power from
        vk = stage_exponent(__uint_as_float(mx << 16));
        vs = ldexpf(1.f, vk);
        // 2^-12 and 2^7 times the first tile's largest (a power of two is 2^7 in a bf16's bits)
        const uint32_t low = mx > 12 << 7 ? mx - (12 << 7) - 1 : 0;
        low2 = low | low << 16;
        top = min(mx + (7 << 7), 0x7f7fu);
      }
      edge(st0, 0);
      convert(st0);
      store(st0, 0, 0);
      load_next(st0, 2);
      edge(st1, min(1, n - 1));
      convert(st1);
      store(st1, 1, 1);
      load_next(st1, 3);
      phase_end();
      if (grp == 1) phase_end();
      qk(0);  // M(0); tiles 0 and 1 are staged above
      phase_end();
      int vrd = 0;  // V slot of tile t
      auto step = [&](int t, Stage& X) SPV_INLINE {  // V(t), M(t + 1); X: tile t + 2
        softmax(t);
        edge(X, min(t + 2, n - 1));
        convert(X);
        window(t + 4);
        phase_end();
        __builtin_amdgcn_s_setprio(1);
        store(X, t & 1, vrd == 0 ? 2 : vrd - 1);
        load(X, min(t + 4, n - 1));
        pv(vrd);
        qk((t + 1) & 1);
        // kAhead operand reads in flight ahead of the matrix instructions (left alone the
        // scheduler keeps two, and each pair waits for its own: 0.83 PFLOP/s; three to
        // eight ahead, 0.86 to 0.91)
        constexpr int kAhead = 4;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < 2 * MT + 4 * KS - kAhead; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * kAhead, 0);
        __builtin_amdgcn_s_setprio(0);
        phase_end();
        vrd = vrd == 2 ? 0 : vrd + 1;
      };
      int t = 0;
      for (; t + 2 < n; t += 2) {
        step(t, st0);
        step(t + 1, st1);
      }
      if (t + 1 < n) {
        step(t, st0);
        ++t;
      }
      softmax(t);
      if constexpr (!kF16 && !kFp8) {
        const bool passed = small || __any((vmax & 0xffffu) > top || (vmax >> 16) > top);
        if (lane == 0) sMax[w] = passed;
      }
      phase_end();
      pv(vrd);
      if (grp == 0) phase_end();
      if constexpr (!kF16 && !kFp8) {
        uint32_t passed = 0;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) passed |= sMax[k];
        if (__builtin_amdgcn_readfirstlane(passed)) return false;
      }
      // (an infinite value and a weight that is 0 in fp16)
      if constexpr (kF16)
        if (__syncthreads_or(sums_not_finite(o)) && __syncthreads_or(values_not_finite(it))) return false;
    }
    write(it, o, m, l, valid, kFp8 ? vref : ldexpf(1.f, -vk));
    return true;
  }

  // The partial rows of a wave of the prefix walk, 16 at a time through memory of its own in
  // LDS: they leave as whole rows (1152 x 2 rows over 2048 keys 20.8 us, 21.9 where each
  // lane stored its own 16 bytes).
  __device__ __forceinline__ void write(const Item& it, const f32x4_t (&o)[MT][NT], const float (&m)[NT],
                                        float (&l)[NT], const bool (&valid)[NT], float post) {
    constexpr int P = D + 4, kQ = D / 4;
    float* const s = reinterpret_cast<float*>(smem) + w * 16 * P;
    __syncthreads();  // the other waves have read their last pages
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] += __shfl_xor(l[nt], 16, 64);
      l[nt] += __shfl_xor(l[nt], 32, 64);
      const int r0 = w * 32 + nt * 16;
      if (g == 0 && valid[nt])
        *reinterpret_cast<float2*>(&p.part_ml[(size_t)(it.part + r0 + i16) * 2]) = make_float2(m[nt], l[nt]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<f32x4_t*>(&s[i16 * P + 16 * mt + 4 * g]) = o[mt][nt] * post;
      __builtin_amdgcn_wave_barrier();
      const int rows = it.rows - r0;
#pragma unroll
      for (int k = 0; k < 16 * kQ / 64; ++k) {
        const int r = (k * 64 + lane) / kQ, q = lane % kQ;
        if (r < rows)
          *reinterpret_cast<f32x4_t*>(&p.part_o[(size_t)(it.part + r0 + r) * D + 4 * q]) =
              *reinterpret_cast<const f32x4_t*>(&s[r * P + 4 * q]);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  __device__ __forceinline__ bool sums_not_finite(const f32x4_t (&o)[MT][NT]) const {  // of the lane
    float z = 0.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) z = fmaf(o[mt][nt][c], 0.f, z);
    return z != z;
  }
  // Whether one of an item's values is not finite: each wave looks through every eighth page.
  __device__ __forceinline__ bool values_not_finite(const Item& it) const {
    constexpr int kPer = 16 / ES;  // elements of a 16-byte piece, of one dim
    constexpr uint32_t kMask = kFp8 ? 0x7fu : kF16 ? 0x7c00u : kF32 ? 0x7f800000u : 0x7f80u;
    const int32_t* table = p.tables + (size_t)it.sid * p.maxb + (it.key0 >> 4);
    bool found = false;
    for (int i = w; it.key0 + 16 * i < it.key1; i += kWaves) {
      const uint8_t* v = page(p.vpool, page_of(safe_id(it, table[i]), it.h));
      const int left = it.key1 - it.key0 - 16 * i;
      for (int c = lane; c < D * ES; c += 64) {
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(v + 16 * c);
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          found |= ((x[e * ES / 4] >> (8 * (e * ES % 4))) & kMask) == kMask && (c * kPer + e) % 16 < left;
      }
    }
    return found;
  }

  // ---- an entry's own keys, and a segment of few rows or in fp32: 32 rows per wave (false: a value
  // is not finite; nothing is written then). nk waves share the
  // rows (8 up to 32 rows, 4 up to 64, 2 up to 128, 1 up to 256) and take every nk-th
  // page straight into operand registers, one page in flight while one is computed;
  // their sums join in LDS.
  // P goes in two halves of bf16 (fp16 pages: of fp16), beside each other in one operand over
  // 16 keys twice: 16 bits of P (22), and values of any size. (fp16 P in one half, over 16 keys
  // once, gave errors of 2.5e-4 against float64 where the output's rounding alone gives 2.1e-4; 64
  // entries of 7 x 16 rows over up to 4000 own keys then took 56.5 us, 58.9 with two.)
  // fp32: v_mfma_f32_16x16x4_f32, four to a 16-byte piece of K or V, whose four elements
  // take turns as the contracted index (the query's and P's, in the same lanes, do the
  // same). At 256 operations a clock and CU the matrix cores take 32 times as long over a
  // page as its 8 KB (head_dim 128) take from the L1, so every wave reads it for itself;
  // K's registers are loaded again while V's are used, and the other way round.
  __device__ __forceinline__ bool pages(const Item& it) {
    using LD = Lds<D>;
    const int nk_log2 = it.rows <= 32 ? 3 : it.rows <= 64 ? 2 : it.rows <= 128 ? 1 : 0, nk = 1 << nk_log2;
    const int kw = w & (nk - 1), r0 = (w >> nk_log2) * 32;
    const int h = __builtin_amdgcn_readfirstlane(it.h), key0 = __builtin_amdgcn_readfirstlane(it.key0),
              key1 = __builtin_amdgcn_readfirstlane(it.key1), start = __builtin_amdgcn_readfirstlane(it.start);
    const int count = (key1 - key0 + 15) >> 4;
    const int32_t* table = p.tables + (size_t)__builtin_amdgcn_readfirstlane(it.sid) * p.maxb + (key0 >> 4);
    const int mine = kw < count ? ((count - 1 - kw) >> nk_log2) + 1 : 0;  // pages kw, kw + nk, ...
    uint4 qf[NT][KS];
    int lim[NT];
    bool valid[NT];
    load_q(it, r0, qf, lim, valid);
    f32x4_t o[MT][NT];
    float m[NT], l[NT], thr[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = -INFINITY;
      l[nt] = 0.f;
      thr[nt] = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    int ids = 0;
    float ksc = 1.f, vsc = 1.f;
    struct Page {
      uint4 k[KS];           // fp8: 8 bytes
      uint32_t v[MT][ES == 4 ? 4 : 2];  // fp8: 4 bytes
    };
    auto load_k = [&](Page& P, int i) SPV_INLINE {
      const int pg = __builtin_amdgcn_readlane(ids, i & 63);
      const uint8_t* K = page(p.kpool, pg) + i16 * D * ES + (kFp8 ? 8 : 16) * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (kFp8) {
          const uint2 x = *reinterpret_cast<const uint2*>(K + 32 * ks);
          P.k[ks] = make_uint4(x.x, x.y, 0u, 0u);
        } else {
          P.k[ks] = *reinterpret_cast<const uint4*>(K + 64 * ks);
        }
      }
    };
    auto load_v = [&](Page& P, int i) SPV_INLINE {
      const int pg = __builtin_amdgcn_readlane(ids, i & 63);
      const uint8_t* V = page(p.vpool, pg) + (i16 * 16 + 4 * g) * ES;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (kFp8) {
          P.v[mt][0] = *reinterpret_cast<const uint32_t*>(V + 256 * mt);
          P.v[mt][1] = 0u;
        } else if constexpr (kF32) {
          const uint4 x = *reinterpret_cast<const uint4*>(V + 1024 * mt);
          P.v[mt][0] = x.x, P.v[mt][1] = x.y, P.v[mt][2] = x.z, P.v[mt][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(V + 512 * mt);
          P.v[mt][0] = x.x, P.v[mt][1] = x.y;
        }
      }
    };
    auto compute = [&](Page& P, int i, int next) SPV_INLINE {  // fp32: `next` is loaded into P
      const int k0 = key0 + 16 * (kw + nk * i);
      f32x4_t sc[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint4 kf = P.k[ks];
        if constexpr (kFp8) {
          const uint32_t a = kf.x, b = kf.y;
          kf = make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true)));
        }
        if constexpr (kF32) {
          const uint32_t k[4] = {kf.x, kf.y, kf.z, kf.w};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t x[4] = {qf[nt][ks].x, qf[nt][ks].y, qf[nt][ks].z, qf[nt][ks].w};
              sc[nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[c]), __uint_as_float(x[c]), sc[nt], 0, 0, 0);
            }
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[nt] = mfma_qk(kf, qf[nt][ks], sc[nt]);
        }
      }
      if constexpr (kF32) load_k(P, next);
      float fv = 1.f;
      if constexpr (kFp8) {
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksc), i & 63));
        fv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vsc), i & 63));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt] *= f;
      }
      if (k0 + 16 > key1 || k0 + 15 > start) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const int key = k0 + 4 * g + jj;
            sc[nt][jj] = key >= key1 || key > lim[nt] ? -INFINITY : sc[nt][jj];
          }
        // Values past the range's end are zero.
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            constexpr uint32_t kMask = kFp8 ? 0xffu : kF32 ? ~0u : 0xffffu;
            const int word = jj * ES / 4, shift = 8 * (jj * ES % 4), key = k0 + 4 * g + jj;
            P.v[mt][word] &= key >= key1 ? ~(kMask << shift) : ~0u;
          }
        }
      }
      bool grow = false;
      float mx[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mx[nt] = fmaxf(max3_raw(sc[nt][0], sc[nt][1], sc[nt][2]), sc[nt][3]);
        grow |= mx[nt] > thr[nt];
      }
      if (__any(grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float a = fmaxf(mx[nt], __shfl_xor(mx[nt], 16, 64));
          a = fmaxf(a, __shfl_xor(a, 32, 64));
          constexpr float kBelow = kF16 ? kShift : 0.f;
          const float m_new = fmaxf(m[nt], a * sl2 - kBelow);
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nt] - m_new);
          l[nt] *= alpha;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) o[mt][nt] *= alpha;
          m[nt] = m_new;
          thr[nt] = (m_new + (kBelow + kSlack)) * inv_sl2;
        }
      }
      uint4 pb[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float mu = m[nt] == -INFINITY ? 0.f : m[nt];
        float e[4];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) e[jj] = __builtin_amdgcn_exp2f(fmaf(sc[nt][jj], sl2, -mu));
        l[nt] += (e[0] + e[1]) + (e[2] + e[3]);
        if constexpr (kF32) {
          pb[nt] = make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3]));
        } else if constexpr (kF16) {
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            hi[k] = pack2_f16(e[2 * k], e[2 * k + 1]);
            const f16x2_t h = __builtin_bit_cast(f16x2_t, hi[k]);
            lo[k] = pack2_f16(e[2 * k] - (float)h[0], e[2 * k + 1] - (float)h[1]);
          }
          pb[nt] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
        } else {
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float a = e[2 * k] * fv, b = e[2 * k + 1] * fv;
            hi[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
            const float ra = a - __uint_as_float(hi[k] << 16), rb = b - __uint_as_float(hi[k] & 0xffff0000u);
            lo[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{ra, rb}, bf16x2_t));
          }
          pb[nt] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (kF32) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t x[4] = {pb[nt].x, pb[nt].y, pb[nt].z, pb[nt].w};
              o[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(P.v[mt][c]), __uint_as_float(x[c]), o[mt][nt], 0, 0, 0);
            }
          continue;
        }
        uint2 v = make_uint2(P.v[mt][0], P.v[mt][1]);
        if constexpr (kFp8) {
          const uint32_t c = v.x;
          v = make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true)));
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (kF16)
            o[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, make_uint4(v.x, v.y, v.x, v.y)),
                                                                __builtin_bit_cast(f16x8_t, pb[nt]), o[mt][nt], 0, 0, 0);
          else
            o[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, make_uint4(v.x, v.y, v.x, v.y)),
                                                                 __builtin_bit_cast(bf16x8_t, pb[nt]), o[mt][nt], 0, 0, 0);
        }
      }
      if constexpr (kF32) {
        __builtin_amdgcn_sched_barrier(0);  // V's registers are free only now
        load_v(P, next);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int base = 0; base < mine; base += 64) {  // 64 of the wave's pages, their ids in the lanes
      const int phys = safe_id(it, table[min(kw + nk * (base + lane), count - 1)]);
      ids = page_of(phys, h);
      if constexpr (kFp8) {
        const float2 s = scales_of(phys);
        ksc = s.x;
        vsc = s.y;
      }
      const int last = min(mine, base + 64) - 1;
      // Every load is unconditional (past the last page it repeats it), so that a page's
      // use waits for its own loads alone.
      Page A;
      load_k(A, base);
      load_v(A, base);
      if constexpr (kF32) {
        for (int i = base; i <= last; ++i) compute(A, i, min(i + 1, last));
      } else {
        Page B;
        for (int i = base;; i += 2) {
          load_k(B, min(i + 1, last));
          load_v(B, min(i + 1, last));
          compute(A, i, 0);
          if (i + 1 > last) break;
          load_k(A, min(i + 2, last));
          load_v(A, min(i + 2, last));
          compute(B, i + 1, 0);
          if (i + 2 > last) break;
        }
      }
    }
    // A value that is not finite must meet neither the P = 0 of rows that do not see it nor a lower
    // half of P (which may be zero or of the other sign): the sums show it as NaN or an infinity,
    // and the any-shape walk takes the item. Keys or queries that are not finite show so, too, but
    // are as right here.
    if (__syncthreads_or(sums_not_finite(o)) && __syncthreads_or(values_not_finite(it))) return false;
    // Join the waves of the same rows: all take the largest m; then every thread adds up
    // four dims of a row over the waves, in their order, half of the dims at a time.
    float2* const sML = reinterpret_cast<float2*>(smem + LD::kJoinRows);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] += __shfl_xor(l[nt], 16, 64);
      l[nt] += __shfl_xor(l[nt], 32, 64);
      if (g == 0) sML[w * 32 + nt * 16 + i16] = make_float2(m[nt], l[nt]);
    }
    __syncthreads();
    const int w0 = w & -nk;  // the first wave of these rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float M = -INFINITY;
      for (int k = 0; k < nk; ++k) M = fmaxf(M, sML[(w0 + k) * 32 + nt * 16 + i16].x);
      const float f = __builtin_amdgcn_exp2f(m[nt] - (M == -INFINITY ? 0.f : M));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][nt] *= f;
    }
    if (tid < it.rows) {
      const int first = (tid >> 5) << nk_log2, r = tid & 31;
      float M = -INFINITY, L = 0.f;
      for (int k = 0; k < nk; ++k) M = fmaxf(M, sML[(first + k) * 32 + r].x);
      const float ref = M == -INFINITY ? 0.f : M;
      for (int k = 0; k < nk; ++k) {
        const float2 x = sML[(first + k) * 32 + r];
        L += x.y * __builtin_amdgcn_exp2f(x.x - ref);
      }
      *reinterpret_cast<float2*>(&p.part_ml[(size_t)(it.part + tid) * 2]) = make_float2(M, L);
    }
    float* const sO = reinterpret_cast<float*>(smem);  // [wave][row][half of the dims], padded
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half) __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT / 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<f32x4_t*>(&sO[(w * 32 + nt * 16 + i16) * LD::kJP + 16 * mt + 4 * g]) =
              o[half * (MT / 2) + mt][nt];
      __syncthreads();
      constexpr int kQ = D / 8;  // pieces of four dims in half a row
      for (int i = tid; i < it.rows * kQ; i += kMfmaThreads) {
        const int r = i / kQ, q = i - r * kQ, first = (r >> 5) << nk_log2;
        f32x4_t x = *reinterpret_cast<const f32x4_t*>(&sO[(first * 32 + (r & 31)) * LD::kJP + 4 * q]);
        for (int k = 1; k < nk; ++k)
          x += *reinterpret_cast<const f32x4_t*>(&sO[((first + k) * 32 + (r & 31)) * LD::kJP + 4 * q]);
        *reinterpret_cast<f32x4_t*>(&p.part_o[(size_t)(it.part + r) * D + half * (D / 2) + 4 * q]) = x;
      }
    }
    return true;
  }
};

template <int D, int KT>
__global__ __launch_bounds__(kMfmaThreads, 2) void shared_mfma_kernel(SharedParams p) {
  static_assert(valu_lds(D) <= Lds<D>::kBytes, "the any-shape walk reuses this memory");
  __shared__ __align__(16) uint8_t smem[Lds<D>::kBytes];
  const int id = blockIdx.x;
  Walk<D, KT> walk(p, smem, threadIdx.x);
  Item it;
  if (id < p.seg_wgs) {
    if (!segment_item(p, id, it)) return;
  } else if (!own_item(p, id - p.seg_wgs, it)) {
    return;
  }
  // A segment of few rows is walked as own keys are, its pages shared out over the waves: 28
  // rows x 2 kv heads of 64 behind 32768 fp16 keys take 10.6 us, 15.3 in a tile of 256 rows
  // (63 x 2 of fp8 13.0 and 18.5; 72 x 2 of 128, bf16, 29.5 and 22.5).
  // Where the tile's staging does not hold its values, they go the same way.
  bool done = false;
  if (KT != SPV_F32 && it.first >= 0 && it.rows > kPagesRows) {
    done = walk.prefix(it);
    if (!done) {  // read again, so that nothing of it stays in registers across the walk
      int again = id;
      asm volatile("" : "+s"(again));
      segment_item(p, again, it);
    }
  }
  if (!done) done = walk.pages(it);
  if (!done) valu_item<Walk<D, KT>::QT, KT, D, kMfmaThreads>(p, it, reinterpret_cast<float*>(smem));
}

// ----------------------------------------------------------------------- join
// LPR lanes per (entry, chunk token, q head), four consecutive dims each (VEC, head_dim =
// 4 LPR), or dims lane + 64 k of any head_dim up to 256; GROUPS such sets of lanes share a
// row's partials. The partials, the prefix's segments in key order and then the entry's own
// ranges, are added in an order that is the row's alone, whatever finished first. With few
// rows latency bounds it: a wave then serves one row, each group reading kJoin partials at
// a time (28 partials of 2016 rows of 64: 5.9 us, one group 10.1; 10 of 1440 rows of 128: 4.9
// and 8.7); with many, the rate of memory (about 5 of 14336 rows: 11.5 us, one group 9.6).
constexpr int kJoin = 4, kFewRows = 8192;
template <int QT, int LPR, int GROUPS, bool VEC>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(SharedParams p) {
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR % GROUPS;
  const long long row = (long long)blockIdx.x * (kThreads / (LPR * GROUPS)) + threadIdx.x / (LPR * GROUPS);
  if (row >= (long long)p.B * p.C * p.Hq) return;
  const int hq = (int)(row % p.Hq), bj = (int)(row / p.Hq), b = bj / p.C, j = bj - b * p.C;
  const int h = hq / p.ratio, r = j * p.ratio + (hq - h * p.ratio);
  const int32_t* e = p.entries + (size_t)b * E_WORDS;
  const int seen = min(max(p.start[b] + p.C, 0), p.max_ctx);
  int np = 0;
  long long pre = 0, step = 0;  // the prefix's partial row of range s: pre + s * step
  if (e[E_SEG] >= 0) {
    const long long R = (long long)e[E_RANK] * p.G + r;
    np = e[E_RANGES];
    step = (long long)e[E_TILES] * p.tile;
    pre = (e[E_SEG] + (long long)h * np * e[E_TILES] + R / p.tile) * p.tile + R % p.tile;
  }
  const int n = np + (seen + p.own_range - 1) / p.own_range;
  const long long own = p.own_part + (long long)(b * p.Hkv + h) * p.own_max * p.G + r;
  float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = group; s0 < n; s0 += GROUPS * kJoin) {  // kJoin partials a round trip
    float2 ml[kJoin];
    float x[kJoin][4];
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      const int s = s0 + k * GROUPS;
      if (s0 + k * GROUPS >= n) {
        ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[k][c] = 0.f;
        continue;
      }
      const size_t at = (size_t)(s < np ? pre + s * step : own + (long long)(s - np) * p.G);
      ml[k] = *reinterpret_cast<const float2*>(&p.part_ml[at * 2]);
      const float* o = p.part_o + at * p.d;
      if constexpr (VEC) {
        const float4 y = *reinterpret_cast<const float4*>(o + 4 * lane);
        x[k][0] = y.x, x[k][1] = y.y, x[k][2] = y.z, x[k][3] = y.w;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[k][c] = lane + 64 * c < p.d ? o[lane + 64 * c] : 0.f;
      }
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) top = fmaxf(top, ml[k].x);
    const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(M - ref);
    M = top;
    L *= keep;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] *= keep;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      if (s0 + k * GROUPS >= n) break;
      const float w = exp2f(ml[k].x - ref);
      L += w * ml[k].y;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] += w * x[k][c];
    }
  }
#pragma unroll
  for (int step = LPR; step < LPR * GROUPS; step *= 2) {  // join the groups
    const float other = __shfl_xor(M, step, 64), top = fmaxf(M, other), ref = top == -INFINITY ? 0.f : top;
    const float mine = exp2f(M - ref), theirs = exp2f(other - ref);
    L = L * mine + __shfl_xor(L, step, 64) * theirs;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = acc[k] * mine + __shfl_xor(acc[k], step, 64) * theirs;
    M = top;
  }
  if (group) return;
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

// ns that a CU takes for a unit of 64 keys with a tile of 256 rows: 8.4 MFLOP at head_dim 128.
long long unit_ns(int kv_dtype, int d, int bs) {
  const bool mfma = bs == 16 && (d == 64 || d == 128);
  return (mfma ? kv_dtype == SPV_F32 ? 14000LL : 2300LL : 70000LL) * d / 128 + 1;
}
// The range of keys per segment, in units: the one for which the workgroups, one for each
// of 256 CUs at a time, end first. A workgroup takes its units and about kFixed ns more to
// start and to end; a partial of 256 rows adds kPartial ns to the whole at head_dim 128, for
// it is written and read again at the rate of memory; and own keys' workgroups (one per
// entry and kv head, that many at least) which find no CU free beside the segments wait for the
// first to end. bf16, 1152 rows x 2 kv heads over 2048 keys: 16 ranges take 28.3 us and
// 8.4 in the join, 8 ranges 20.8 and 5.7; 1008 rows x 2 over 32768 keys of fp8 with 32 such
// workgroups: 31 ranges take 49.1 and 11.7, 27 ranges 43.4 and 10.1.
// fp32 tiles may have fewer rows, where the matrix cores of more CUs are worth reading the
// keys again: ten entries of 30 rows x 2 behind three prefixes of up to 1501 keys take 19.1 us in
// tiles of 64 rows, 23.3 in tiles of 256 (32 such entries behind 4096 keys 59.9 and 68.9).
constexpr int kCUs = 256, kFixed = 9000, kPartial = 110;
long long best_range(const std::vector<long long>& tiles, const std::vector<long long>& units, long long own,
                     long long unit, int d, int rows, long long* range_out) {
  long long most = 1, best = 1, least = -1;
  for (long long u : units) most = std::max(most, u);
  // ceil(most / k) for every number of ranges k: no other length cuts the longest prefix evenly
  for (long long k = 1; k <= most; ++k) {
    const long long range = (most + k - 1) / k;
    long long n = 0;
    for (size_t g = 0; g < units.size(); ++g) n += tiles[g] * ((units[g] + range - 1) / range);
    const long long rounds = (n + kCUs - 1) / kCUs;
    const long long late = n + own > rounds * kCUs ? kFixed : 0;
    const long long time =
        rounds * (range * unit * rows / kTile + kFixed) + late + n * kPartial * d / 128 * rows / kTile;
    if (least < 0 || time < least) {
      least = time;
      best = range;
    }
    if (n > 4 * kCUs && k > 1) break;  // more, shorter segments only add to the fixed part
  }
  *range_out = best;
  return least;
}

int make_plan(std::vector<int32_t>& plan, const int32_t* ids, const int32_t* lens, int B, int C, int Hq, int Hkv, int d,
              int bs, int kv_dtype) {
  const long long G = (long long)C * (Hq / Hkv);
  std::vector<Group> groups;
  std::map<std::pair<int32_t, int32_t>, size_t> index;
  std::vector<int32_t> entries(E_WORDS * (size_t)B, 0), of(B, -1), members, segs;
  for (int b = 0; b < B; ++b) {
    if (ids[b] < -1 || lens[b] < 0) return SPV_ERR_ARG;
    entries[E_WORDS * (size_t)b + E_SEG] = -1;
    if (ids[b] < 0 || lens[b] == 0) continue;
    const size_t g = index.emplace(std::make_pair(ids[b], lens[b]), groups.size()).first->second;
    if (g == groups.size()) groups.push_back({ids[b], lens[b], {}});
    entries[E_WORDS * (size_t)b + E_RANK] = (int)groups[g].members.size();
    of[b] = (int)g;
    groups[g].members.push_back(b);
  }
  std::vector<long long> tiles, units;
  long long maxp = 0, range = 1, least = -1;
  int tile = kTile;
  for (const Group& x : groups) {
    units.push_back((x.len + kUnit - 1LL) / kUnit);
    maxp = std::max<long long>(maxp, x.len);
  }
  for (int rows = kTile; rows >= (kv_dtype == SPV_F32 ? kPagesRows : kTile); rows /= 2) {
    std::vector<long long> cut, all;
    for (const Group& x : groups) {
      cut.push_back(((long long)x.members.size() * G + rows - 1) / rows);
      all.push_back(cut.back() * Hkv);
    }
    long long best = 1;
    const long long time = best_range(all, units, (long long)B * Hkv, unit_ns(kv_dtype, d, bs), d, rows, &best);
    if (least < 0 || time < least) {
      least = time;
      range = best;
      tile = rows;
      tiles = cut;
    }
  }
  long long nseg = 0;
  for (size_t g = 0; g < groups.size(); ++g) {
    const Group& x = groups[g];
    // equal ranges, of whole units
    const long long ranges = (units[g] + range - 1) / range, per = (units[g] + ranges - 1) / ranges;
    const long long used = (units[g] + per - 1) / per, rows = (long long)x.members.size() * G;
    if ((nseg + tiles[g] * Hkv * used) > 0x7fffffffLL / tile) return SPV_ERR_UNSUPPORTED;
    for (int h = 0; h < Hkv; ++h)
      for (long long s = 0; s < used; ++s)
        for (long long t = 0; t < tiles[g]; ++t) {
          const int32_t w[S_WORDS] = {x.sid, x.len, h, (int32_t)members.size(), (int32_t)(t * tile),
                                      (int32_t)std::min<long long>(tile, rows - t * tile), (int32_t)(s * per * kUnit),
                                      (int32_t)std::min<long long>((s + 1) * per * kUnit, x.len)};
          segs.insert(segs.end(), w, w + S_WORDS);
        }
    for (int b : x.members) {
      int32_t* const e = &entries[E_WORDS * (size_t)b];
      e[E_SEG] = (int32_t)nseg;
      e[E_TILES] = (int32_t)tiles[g];
      e[E_RANGES] = (int32_t)used;
    }
    nseg += tiles[g] * Hkv * used;
    members.insert(members.end(), x.members.begin(), x.members.end());
  }
  plan.assign(PH_WORDS, 0);
  plan[PH_MAGIC] = kPlanMagic;
  plan[PH_B] = B;
  plan[PH_C] = C;
  plan[PH_HQ] = Hq;
  plan[PH_HKV] = Hkv;
  plan[PH_BS] = bs;
  plan[PH_NSEG] = (int32_t)nseg;
  plan[PH_MAXP] = (int32_t)maxp;
  plan[PH_TILE] = tile;
  plan[PH_OWN] = kv_dtype == SPV_F32 ? 64 : 256;
  auto add = [&](int word, const std::vector<int32_t>& v) {
    while (plan.size() % 16) plan.push_back(0);
    plan[word] = (int32_t)plan.size();
    plan.insert(plan.end(), v.begin(), v.end());
  };
  add(PH_SEGS, segs);
  add(PH_MEMBERS, members);
  add(PH_ENTRIES, entries);
  plan[PH_INTS] = (int32_t)plan.size();
  return SPV_OK;
}

// The entries' own ranges for contexts up to max_ctx: as many as make about 256
// workgroups (one for each CU), none shorter than PH_OWN keys: 256 (four waves with four
// pages each), 64 in fp32, where a page takes a wave sixteen times as long. Where the
// prefixes' segments leave CUs free, half of that (24 x 2 rows of own and prefix, bf16: 13.0
// us, 15.4 with 256 keys); and up to twice as long where the CUs beside them then do (192 x 2
// rows 21.2 us, 24.8 where some wait; 12 entries of 30 x 2 rows in fp32 19.1 and 26.9).
// Long contexts of fewer entries and heads than CUs are cut into up to 1024, of 4 PH_OWN keys at
// least, so that the longest do not end alone: 64 entries x 2 kv heads of 16 to 4000 keys behind
// 2000 take 73.5 us, 95.5 with 256 (200 entries of up to 3000 behind 500 149.7 and 137.3).
void own_ranges(const int32_t* plan, int max_ctx, int* range, int* count) {
  const int bs = plan[PH_BS];
  const long long G = (long long)plan[PH_C] * (plan[PH_HQ] / plan[PH_HKV]), least = plan[PH_OWN];
  const long long wgs = (long long)plan[PH_B] * plan[PH_HKV] * ((G + kOwnRows - 1) / kOwnRows);
  long long all = std::min(kCUs / wgs, max_ctx / least);
  if (wgs < kCUs) all = std::max(all, std::min(4 * kCUs / wgs, max_ctx / (4 * least)));
  const long long beside = std::min((kCUs - std::min(kCUs, plan[PH_NSEG])) / wgs, max_ctx / (least / 2));
  const long long want = std::max(1LL, 2 * beside >= all ? beside : all);
  const long long keys = (max_ctx + want - 1) / want;
  *range = (int)((keys + bs - 1) / bs * bs);
  *count = (max_ctx + *range - 1) / *range;
}

long long part_rows(const int32_t* plan, int max_ctx) {
  int range, count;
  own_ranges(plan, max_ctx, &range, &count);
  const long long G = (long long)plan[PH_C] * (plan[PH_HQ] / plan[PH_HKV]);
  return (long long)plan[PH_NSEG] * plan[PH_TILE] + (long long)plan[PH_B] * plan[PH_HKV] * count * G;
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
  hipLaunchKernelGGL((shared_mfma_kernel<D, KT>), dim3((unsigned)grid), dim3(kMfmaThreads), 0, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

template <int QT, int LPR, int GROUPS, bool VEC>
int launch_join(const SharedParams& p, hipStream_t s) {
  const long long rows = (long long)p.B * p.C * p.Hq, per = kThreads / (LPR * GROUPS);
  hipLaunchKernelGGL((shared_join_kernel<QT, LPR, GROUPS, VEC>), dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads),
                     0, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

template <int QT>
int launch(const SharedParams& p, int kv_dtype, hipStream_t s) {
  const long long grid = p.seg_wgs + (long long)p.B * p.Hkv * p.own_tiles * p.own_max;
  int rc;
  // The matrix kernels apply the scale inside the exponent, to maxima of raw scores.
  // They count pages in 31 bits and load 16 bytes at a time.
  const auto aligned = [](const void* x) { return (uintptr_t)x % 16 == 0; };
  const bool mfma = aligned(p.q) && aligned(p.kpool) && aligned(p.vpool) &&
                    (long long)(p.layer + 1) * p.cap * p.Hkv < (1LL << 31) && p.bs == 16 &&
                    (p.d == 64 || p.d == 128) && p.scale_log2 > 0.f && p.scale_log2 < INFINITY &&
                    ((QT == SPV_BF16 && kv_dtype == SPV_FP8E4M3) || QT == kv_dtype);
  if (mfma) {
    if constexpr (QT == SPV_BF16) {
      if (kv_dtype == SPV_BF16) rc = p.d == 64 ? launch_mfma<64, SPV_BF16>(p, grid, s) : launch_mfma<128, SPV_BF16>(p, grid, s);
      else rc = p.d == 64 ? launch_mfma<64, SPV_FP8E4M3>(p, grid, s) : launch_mfma<128, SPV_FP8E4M3>(p, grid, s);
    } else {
      rc = p.d == 64 ? launch_mfma<64, QT>(p, grid, s) : launch_mfma<128, QT>(p, grid, s);
    }
  } else switch (kv_dtype) {
    case SPV_F32: rc = launch_valu<QT, SPV_F32>(p, grid, s); break;
    case SPV_BF16: rc = launch_valu<QT, SPV_BF16>(p, grid, s); break;
    case SPV_F16: rc = launch_valu<QT, SPV_F16>(p, grid, s); break;
    default: rc = launch_valu<QT, SPV_FP8E4M3>(p, grid, s); break;
  }
  if (rc != SPV_OK) return rc;
  const bool few = (long long)p.B * p.C * p.Hq < kFewRows;
  if (!aligned(p.out)) return launch_join<QT, 64, 1, false>(p, s);
  if (p.d == 128) return few ? launch_join<QT, 32, 2, true>(p, s) : launch_join<QT, 32, 1, true>(p, s);
  if (p.d == 64) return few ? launch_join<QT, 16, 4, true>(p, s) : launch_join<QT, 16, 1, true>(p, s);
  return launch_join<QT, 64, 1, false>(p, s);
}

}  // namespace

extern "C" {

int64_t spv_shared_attn_plan(const int32_t* prefix_ids, const int32_t* prefix_lens, int32_t B, int32_t C,
                             int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                             int kv_dtype, int32_t* plan, int64_t plan_ints) {
  if (!prefix_ids || !prefix_lens || B < 1 || B > 65535 || C < 1 || num_kv_heads < 1 ||
      num_q_heads < num_kv_heads || num_q_heads % num_kv_heads || block_size < 1 || head_dim < 1 ||
      head_dim > kMaxD || dtype_size(kv_dtype) == 0 ||
      (long long)C * num_q_heads > (1 << 20) || (long long)B * C * num_q_heads > (1LL << 30))
    return SPV_ERR_ARG;
  try {
    std::vector<int32_t> p;
    const int rc = make_plan(p, prefix_ids, prefix_lens, B, C, num_q_heads, num_kv_heads, head_dim, block_size, kv_dtype);
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
  if (workspace_bytes < spv_shared_attn_workspace_bytes(h, head_dim, max_ctx) || (uintptr_t)workspace % 16)
    return SPV_ERR_WORKSPACE;
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
  p.segs = plan + h[PH_SEGS];
  p.members = plan + h[PH_MEMBERS];
  p.entries = plan + h[PH_ENTRIES];
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
  p.tile = h[PH_TILE];
  p.nseg = h[PH_NSEG];
  p.seg_wgs = (p.nseg + 7) / 8 * 8;
  p.max_ctx = max_ctx;
  own_ranges(h, max_ctx, &p.own_range, &p.own_max);
  p.own_tiles = (p.G + kOwnRows - 1) / kOwnRows;
  p.own_part = (long long)h[PH_NSEG] * h[PH_TILE];
  const long long rows = part_rows(h, max_ctx);
  // both grids: at most 2^32 threads
  const long long own = (long long)B * num_kv_heads * p.own_tiles * p.own_max;
  if (p.seg_wgs + own > (1LL << 22) || (long long)B * C * num_q_heads > (1LL << 23)) return SPV_ERR_UNSUPPORTED;
  p.part_ml = static_cast<float*>(workspace);
  p.part_o = p.part_ml + ml_floats((size_t)rows);
  p.scale_log2 = scale * kLog2e;
  hipStream_t s = (hipStream_t)stream;
  if (q_dtype == SPV_F32) return launch<SPV_F32>(p, kv_dtype, s);
  if (q_dtype == SPV_BF16) return launch<SPV_BF16>(p, kv_dtype, s);
  return launch<SPV_F16>(p, kv_dtype, s);
}

}  // extern "C"
