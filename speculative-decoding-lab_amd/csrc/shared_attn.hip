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
// end to end -- (member, chunk token, head of the group) -- and cut into tiles; an
// item of the work list is one tile over one range of the prefix. An entry's
// own keys are walked by further items, one per (entry, kv head, range). Every
// item leaves a partial; a second launch joins each row's. The items are
// listed on the host (the prefixes and their lengths change when a request is
// admitted, not between rounds); the entries' own lengths are read on the
// device.
#include <math.h>

#include <algorithm>
#include <map>
#include <utility>
#include <vector>

#include "spv_common.h"

using namespace spv;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The plan: a header, the groups, the entries in group order, each entry's
// place, the items.
enum : int {
  PH_MAGIC = 0,
  PH_INTS,     // length of the plan
  PH_B,
  PH_C,
  PH_HQ,
  PH_HKV,
  PH_BS,
  PH_TILE,     // rows of an item's tile
  PH_NG,       // groups
  PH_ITEMS,
  PH_PARTS,    // partial rows of all items
  PH_MAXP,     // longest prefix
  PH_GROUPS,   // offsets of the sections
  PH_MEMBERS,
  PH_ENTRIES,
  PH_LIST,
  PH_WORDS
};
constexpr int kPlanMagic = 0x53505231;
enum : int { G_SID = 0, G_LEN, G_FIRST, G_COUNT, G_SPLITS, G_RANGE, G_PART, G_WORDS = 8 };  // G_RANGE: keys per split
enum : int { E_GROUP = 0, E_RANK, E_WORDS };
enum : int { I_GROUP = 0, I_HEAD, I_TILE, I_SPLIT, I_WORDS };

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
  int tile, items;         // prefix items
  int own_range, own_max;  // keys per own range (a multiple of the block size), ranges per entry at most
  int max_ctx;
  long long own_part;      // first partial row of the own ranges
  float scale_log2;
};

// One item: rows [row0, row0 + rows) of a group's (or one entry's) row order
// over keys [key0, key1) of one sequence.
struct Item {
  int group, sid, b, h, row0, rows, key0, key1, first, limit;  // limit: keys row j sees are <= limit + j
  long long part;
};

__device__ __forceinline__ void flag_bad_read(const SharedParams& p, int b) {
  if (p.ctr) p.ctr[CTR_BAD_READ] = b + 1;
}

// Item `id` of the launch; false where it has no keys.
__device__ __forceinline__ bool item_of(const SharedParams& p, int id, Item& it) {
  if (id < p.items) {
    const int32_t* l = p.plan + p.plan[PH_LIST] + (size_t)id * I_WORDS;
    const int32_t* g = p.plan + p.plan[PH_GROUPS] + (size_t)l[I_GROUP] * G_WORDS;
    const int total = g[G_COUNT] * p.G;
    it.group = l[I_GROUP];
    it.sid = g[G_SID];
    it.h = l[I_HEAD];
    it.first = p.plan[PH_MEMBERS] + g[G_FIRST];
    it.b = p.plan[it.first];
    it.row0 = l[I_TILE] * p.tile;
    it.rows = min(p.tile, total - it.row0);
    it.key0 = l[I_SPLIT] * g[G_RANGE];
    it.key1 = min(it.key0 + g[G_RANGE], g[G_LEN]);
    it.limit = 0x3fffffff;
    it.part = g[G_PART] + ((long long)it.h * g[G_SPLITS] + l[I_SPLIT]) * total + it.row0;
    if (threadIdx.x == 0 && p.lens && p.lens[it.sid] < g[G_LEN]) flag_bad_read(p, it.b);
    return true;
  }
  const int o = id - p.items;
  const int s = o % p.own_max, bh = o / p.own_max;
  it.group = -1;
  it.b = bh / p.Hkv;
  it.h = bh - it.b * p.Hkv;
  it.sid = p.seq_ids[it.b];
  it.limit = p.start[it.b];
  const int L = it.limit + p.C, seen = min(max(L, 0), p.max_ctx);
  if (threadIdx.x == 0 && s == 0 && it.h == 0 && (it.limit < 0 || L > p.max_ctx || (p.lens && p.lens[it.sid] < L)))
    flag_bad_read(p, it.b);
  it.row0 = 0;
  it.rows = p.G;
  it.first = 0;
  it.key0 = s * p.own_range;
  it.key1 = min(it.key0 + p.own_range, seen);
  it.part = p.own_part + ((long long)bh * p.own_max + s) * p.G;
  return it.key0 < it.key1;
}

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
// later positions hold (infinities, NaN) never reaches it.
constexpr int kThreads = 256;
constexpr int kRows = 64;
constexpr int kKeys = 16;

template <int QT, int KT>
__global__ __launch_bounds__(kThreads) void shared_valu_kernel(SharedParams p) {
  extern __shared__ float smem[];
  Item it;
  if (!item_of(p, blockIdx.x, it)) return;
  const int d = p.d;
  float* Qs = smem;                    // [64][d], in log2 units
  float* Ks = Qs + kRows * d;          // [16][d]
  float* Vs = Ks + kKeys * d;          // [16][d]
  float* Ps = Vs + kKeys * d;          // [64][17]
  float* Ms = Ps + kRows * (kKeys + 1);
  float* Ls = Ms + kRows;
  float* As = Ls + kRows;
  int* Lim = reinterpret_cast<int*>(As + kRows);  // last key a row sees
  for (int r0 = 0; r0 < it.rows; r0 += kRows) {
    const int nr = min(kRows, it.rows - r0);
    for (int i = threadIdx.x; i < nr * d; i += kThreads) {
      const int rr = i / d, e = i - rr * d;
      int b, j, hq;
      row_at(p, it, it.row0 + r0 + rr, b, j, hq);
      Qs[rr * d + e] = load_elem<QT>(p.q, (((size_t)b * p.C + j) * p.Hq + hq) * d + e) * p.scale_log2;
      if (e == 0) Lim[rr] = it.group >= 0 ? it.limit : it.limit + j;
    }
    if (threadIdx.x < kRows) {
      Ms[threadIdx.x] = -INFINITY;
      Ls[threadIdx.x] = 0.f;
    }
    constexpr int kMaxO = kRows * 256 / kThreads;
    float o[kMaxO];
#pragma unroll
    for (int k = 0; k < kMaxO; ++k) o[k] = 0.f;
    __syncthreads();
    for (int t0 = it.key0; t0 < it.key1; t0 += kKeys) {
      const int nt = min(kKeys, it.key1 - t0);
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
        Ks[tt * d + e] = kv;
        Vs[tt * d + e] = vv;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < nr * kKeys; i += kThreads) {
        const int rr = i / kKeys, tt = i - rr * kKeys;
        float sc = -INFINITY;
        if (tt < nt && t0 + tt <= Lim[rr]) {
          float acc = 0.f;
          for (int e = 0; e < d; ++e) acc = fmaf(Qs[rr * d + e], Ks[tt * d + e], acc);
          sc = acc;
        }
        Ps[rr * (kKeys + 1) + tt] = sc;
      }
      __syncthreads();
      if ((int)threadIdx.x < nr) {
        const int rr = threadIdx.x;
        float* P = Ps + rr * (kKeys + 1);
        float mx = Ms[rr];
        for (int tt = 0; tt < kKeys; ++tt) mx = fmaxf(mx, P[tt]);
        const float ref = mx == -INFINITY ? 0.f : mx;  // a row without a finite score yet: its P are 0 (or NaN)
        const float alpha = exp2f(Ms[rr] - ref);
        float sum = 0.f;
        for (int tt = 0; tt < kKeys; ++tt) {
          P[tt] = exp2f(P[tt] - ref);
          sum += P[tt];
        }
        Ls[rr] = Ls[rr] * alpha + sum;
        Ms[rr] = mx;
        As[rr] = alpha;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kMaxO; ++k) {
        const int el = threadIdx.x + k * kThreads;
        if (el < nr * d) {
          const int rr = el / d, e = el - rr * d;
          float acc = o[k] * As[rr];
          const int n = min(nt, Lim[rr] - t0 + 1);
          for (int tt = 0; tt < n; ++tt) acc = fmaf(Ps[rr * (kKeys + 1) + tt], Vs[tt * d + e], acc);
          o[k] = acc;
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kMaxO; ++k) {
      const int el = threadIdx.x + k * kThreads;
      if (el < nr * d) {
        const int rr = el / d, e = el - rr * d;
        const size_t row = (size_t)(it.part + r0 + rr);
        p.part_o[row * d + e] = o[k];
        if (e == 0) *reinterpret_cast<float2*>(&p.part_ml[row * 2]) = make_float2(Ms[rr], Ls[rr]);
      }
    }
    __syncthreads();
  }
}

// ----------------------------------------------------------------------- join
// One wave per (entry, chunk token, q head): the row's partials, the prefix's
// ranges then its own, in that order whatever finished first.
template <int QT>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(SharedParams p) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= (long long)p.B * p.C * p.Hq) return;
  const int hq = (int)(row % p.Hq), bj = (int)(row / p.Hq), b = bj / p.C, j = bj - b * p.C;
  const int h = hq / p.ratio, r = j * p.ratio + hq % p.ratio;
  const int32_t* e = p.plan + p.plan[PH_ENTRIES] + (size_t)b * E_WORDS;
  int np = 0;
  long long pre = 0, step = 0;  // the prefix's partial of range s: row pre + s * step
  if (e[E_GROUP] >= 0) {
    const int32_t* g = p.plan + p.plan[PH_GROUPS] + (size_t)e[E_GROUP] * G_WORDS;
    np = g[G_SPLITS];
    step = (long long)g[G_COUNT] * p.G;
    pre = g[G_PART] + (long long)h * np * step + (long long)e[E_RANK] * p.G + r;
  }
  const int seen = min(max(p.start[b] + p.C, 0), p.max_ctx);
  const int no = (seen + p.own_range - 1) / p.own_range;
  const long long own = p.own_part + ((long long)(b * p.Hkv + h) * p.own_max) * p.G + r;
  auto part = [&](int s) { return (size_t)(s < np ? pre + s * step : own + (long long)(s - np) * p.G); };
  float M = -INFINITY;
  for (int s = lane; s < np + no; s += 64) M = fmaxf(M, p.part_ml[part(s) * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  const float ref = M == -INFINITY ? 0.f : M;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, L = 0.f;  // head_dim <= 256: dims lane + 64 k
  for (int s = 0; s < np + no; ++s) {
    const size_t at = part(s);
    const float2 ml = *reinterpret_cast<const float2*>(&p.part_ml[at * 2]);
    const float w = exp2f(ml.x - ref);
    L += w * ml.y;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane + 64 * k < p.d) acc[k] += w * p.part_o[at * p.d + lane + 64 * k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < p.d) store_elem<QT>(p.out, (size_t)row * p.d + lane + 64 * k, acc[k] / L);
}

// ----------------------------------------------------------------------- plan
struct Group {
  int sid, len;
  std::vector<int> members;
};

int make_plan(std::vector<int32_t>& plan, const int32_t* ids, const int32_t* lens, int B, int C, int Hq, int Hkv,
              int bs) {
  const int G = C * (Hq / Hkv), tile = 64;
  std::vector<Group> groups;
  std::map<std::pair<int32_t, int32_t>, size_t> index;
  std::vector<int32_t> entries(2 * (size_t)B);
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
  // Ranges of the prefixes: about 1,024 items, none shorter than 64 keys.
  long long units = 0;  // tiles x keys
  for (const Group& g : groups)
    units += (long long)Hkv * ((g.members.size() * (long long)G + tile - 1) / tile) * g.len;
  const long long range = std::max(64LL, (units + 1023) / 1024);
  std::vector<int32_t> gw, mw, iw;
  long long part = 0, maxp = 0;
  for (size_t g = 0; g < groups.size(); ++g) {
    const Group& x = groups[g];
    const long long rows = (long long)x.members.size() * G, tiles = (rows + tile - 1) / tile;
    const long long want = std::max(1LL, (x.len + range - 1) / range);
    long long keys = (x.len + want - 1) / want;
    keys = (keys + bs - 1) / bs * bs;
    const long long splits = (x.len + keys - 1) / keys;
    const int32_t w[G_WORDS] = {x.sid, x.len, (int32_t)mw.size(), (int32_t)x.members.size(), (int32_t)splits,
                                (int32_t)keys, (int32_t)part, 0};
    gw.insert(gw.end(), w, w + G_WORDS);
    mw.insert(mw.end(), x.members.begin(), x.members.end());
    for (int s = 0; s < (int)splits; ++s)
      for (int t = 0; t < (int)tiles; ++t)
        for (int h = 0; h < Hkv; ++h) {
          const int32_t i[I_WORDS] = {(int32_t)g, h, t, s};
          iw.insert(iw.end(), i, i + I_WORDS);
        }
    part += rows * Hkv * splits;
    maxp = std::max<long long>(maxp, x.len);
    if (part > 0x7fffffffLL) return SPV_ERR_UNSUPPORTED;
  }
  plan.assign(PH_WORDS, 0);
  plan[PH_MAGIC] = kPlanMagic;
  plan[PH_B] = B;
  plan[PH_C] = C;
  plan[PH_HQ] = Hq;
  plan[PH_HKV] = Hkv;
  plan[PH_BS] = bs;
  plan[PH_TILE] = tile;
  plan[PH_NG] = (int32_t)groups.size();
  plan[PH_ITEMS] = (int32_t)(iw.size() / I_WORDS);
  plan[PH_PARTS] = (int32_t)part;
  plan[PH_MAXP] = (int32_t)maxp;
  auto add = [&](int word, const std::vector<int32_t>& v) {
    plan[word] = (int32_t)plan.size();
    plan.insert(plan.end(), v.begin(), v.end());
  };
  add(PH_GROUPS, gw);
  add(PH_MEMBERS, mw);
  add(PH_ENTRIES, entries);
  add(PH_LIST, iw);
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
  return plan[PH_PARTS] + (long long)plan[PH_B] * plan[PH_HKV] * count * G;
}

// Floats of the (m, l) pairs at the workspace's head: whole 16-byte pieces, so that the rows behind them are aligned.
size_t ml_floats(size_t rows) { return (2 * rows + 3) / 4 * 4; }

template <int QT, int KT>
int launch_valu(const SharedParams& p, long long grid, hipStream_t s) {
  const size_t smem = (size_t)((kRows + 2 * kKeys) * p.d + kRows * (kKeys + 1) + 4 * kRows) * sizeof(float);
  if (smem > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(&shared_valu_kernel<QT, KT>),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != hipSuccess)
    return SPV_ERR_LAUNCH;
  hipLaunchKernelGGL((shared_valu_kernel<QT, KT>), dim3((unsigned)grid), dim3(kThreads), smem, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
}

template <int QT>
int launch(const SharedParams& p, int kv_dtype, hipStream_t s) {
  const long long grid = p.items + (long long)p.B * p.Hkv * p.own_max;
  int rc;
  switch (kv_dtype) {
    case SPV_F32: rc = launch_valu<QT, SPV_F32>(p, grid, s); break;
    case SPV_BF16: rc = launch_valu<QT, SPV_BF16>(p, grid, s); break;
    case SPV_F16: rc = launch_valu<QT, SPV_F16>(p, grid, s); break;
    default: rc = launch_valu<QT, SPV_FP8E4M3>(p, grid, s); break;
  }
  if (rc != SPV_OK) return rc;
  const long long rows = (long long)p.B * p.C * p.Hq;
  hipLaunchKernelGGL(shared_join_kernel<QT>, dim3((unsigned)((rows + kThreads / 64 - 1) / (kThreads / 64))),
                     dim3(kThreads), 0, s, p);
  SPV_CHECK_LAUNCH();
  return SPV_OK;
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
  p.tile = h[PH_TILE];
  p.items = h[PH_ITEMS];
  p.max_ctx = max_ctx;
  own_ranges(h, max_ctx, &p.own_range, &p.own_max);
  p.own_part = h[PH_PARTS];
  const long long rows = part_rows(h, max_ctx);
  if (p.items + (long long)B * num_kv_heads * p.own_max > (1LL << 23)) return SPV_ERR_UNSUPPORTED;  // the grid
  p.part_ml = static_cast<float*>(workspace);
  p.part_o = p.part_ml + ml_floats((size_t)rows);
  p.scale_log2 = scale * kLog2e;
  hipStream_t s = (hipStream_t)stream;
  if (q_dtype == SPV_F32) return launch<SPV_F32>(p, kv_dtype, s);
  if (q_dtype == SPV_BF16) return launch<SPV_BF16>(p, kv_dtype, s);
  return launch<SPV_F16>(p, kv_dtype, s);
}

}  // extern "C"
