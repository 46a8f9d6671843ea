// window_attn.cu -- paged attention through a sliding window with sinks: the query at position p
// sees key j when j <= p and (j > p - window or j < sinks).  The mask beside those of
// crates/higgs-models/src/utils.rs:64-125; q, K / V pages and rounding points as in
// higgs_paged_attention (utils.rs:45-60).
//
// Pages wholly behind the window and past the sinks are neither looked up nor read, so a host may
// free them.  Rows whose position is negative (a query batch longer than its sequence) see nothing
// and give zeros.
//
// Decode kernel (few query rows per kv head).  A CTA takes a split of the visible pages of one
// (sequence, kv head, tile of 8 query rows = tokens x the G heads of the kv head), its 4 warps
// alternate over the pages.  The page's 16 keys are the MMA's 16 rows and the query rows its 8
// columns, so G = 4 heads waste half of the tile and not three quarters of it:
//   S^T = K Q^T     A = K, 16 keys x 16 of d,     B = Q^T
//   O^T += V^T P^T  A = V^T, 16 of d x 16 keys,   B = P^T
// Both A operands come straight from global memory, 16 bytes per lane and load, with no shared
// memory between: the sum over d may run in any order, so a lane's 16 bytes of a K row serve two
// MMA steps (Q is laid out the same way); and the rows of O^T may be any d, so a lane loads 16
// bytes of each of its 4 keys of V and pairs the keys with PRMT.  P^T goes from the accumulator's
// layout to B's by an 8x8 transpose in registers (movmatrix), as bf16 hi + lo halves: 16 bits of
// the weights, as in the other decode kernels.  The running maximum moves only when a score
// exceeds it by 2^kSlack.  Tiles of 16 or 32 query rows (more columns per page load) measured
// slower for six-token verifies, 8 sequences of 1000 visible keys 15.9 and 19.0 against 13.1 us:
// the warps' chains get longer while the GPU is far from full.
// Bound: HBM, 4 * D bytes per visible key and kv head.  B200, D = 128, 8 kv heads: 32 sequences of
// 4100 visible keys (537 MB) 90.7 us = 5.93 TB/s, 0.92 of a copy; one sequence of 1028 keys 6.6 us,
// bound by its chain of launch, length, page id, page, merge, counter and join.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"

namespace higgs {
namespace {

constexpr int kWinThreads = 128;
constexpr int kWinWarps = kWinThreads / 32;
constexpr int kWinCounterBytes = 16384;
constexpr int kRows = 8;  // query rows of a tile: the columns of the MMA
constexpr int kMaxSplits = 64;
constexpr int kCtasPerSm128 = 3, kCtasPerSm64 = 5;  // resident at once (registers)
constexpr float kSlack = 8.0f;  // log2

struct WinArgs {
  const uint16_t* q;
  const uint16_t* kc;
  const uint16_t* vc;
  int64_t page_stride, head_stride;
  const int32_t* bt;
  int max_blocks;
  const int32_t* seq_lens;
  int Lq, Hq, Hkv, G, window, sinks;
  uint32_t inv_G;  // 2^32 / G, rounded up
  float scale_log2;
  uint16_t* out;
  int splits, tiles;
  int* counters;  // [B * Hkv * tiles] splits done: zero before the launch, zero after it
  float* part;      // [pairs][splits][rows of a tile][D]: sums of the splits
  float2* part_ml;  // [pairs][splits][rows of a tile]: their maxima and norms
};

// The visible pages of a tile of queries at positions p_lo .. p_hi: the sinks' pages, then the
// window's.  Page i of them is page(i) of the sequence.
struct Visible {
  int lo, sink_pages, n;  // lo: first key of the window of p_lo
  __device__ Visible(int p_lo, int p_hi, int window, int sinks) {
    lo = max(0, p_lo - window + 1);
    const int sink_keys = min(sinks, p_hi + 1);
    sink_pages = min((sink_keys + 15) >> 4, lo >> 4);
    n = p_hi < 0 ? 0 : sink_pages + (p_hi >> 4) - (lo >> 4) + 1;
  }
  __device__ int page(int i) const { return i < sink_pages ? i : i - sink_pages + (lo >> 4); }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t part4(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

__device__ __forceinline__ uint4 ldg16_if(const uint16_t* p, bool ok) {
  return ok ? ldg_stream_u4(p) : make_uint4(0, 0, 0, 0);
}

// Row r of kv head h's tokens x heads as (query token, query head) of the call: r / G by a
// multiplication (exact while r * G < 2^32, which the host checks).
struct Row {
  int t, head;
  __device__ Row(const WinArgs& a, int h, int r) {
    t = a.G == 1 ? r : (int)__umulhi((uint32_t)r, a.inv_G);
    head = h * a.G + r - t * a.G;
  }
};

// 2^x, results below 2^-126 flushed to zero
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D>
__global__ void __launch_bounds__(kWinThreads) window_decode_kernel(WinArgs a) {
  constexpr int KC = D / 32;     // 16-byte chunks of a K row per lane
  constexpr int VC = D / 64;     // 16-byte chunks of a V row per lane
  constexpr int MT = D / 16;     // 16-row tiles of O^T
  constexpr int QS = D + 8;      // padded rows of Q and of O in shared memory
  constexpr int OS = D + 4;
  __shared__ __align__(16) uint16_t qs[kRows * QS];
  __shared__ __align__(16) float sm_o[kWinWarps * kRows * OS];
  __shared__ float2 sm_ml[kWinWarps][kRows];  // maximum, norm
  __shared__ float sm_f[kWinWarps][kRows];
  __shared__ int is_last;
  const int split = blockIdx.x, h = blockIdx.y / a.tiles, tile = blockIdx.y - h * a.tiles, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = a.G * a.Lq, r0 = tile * kRows, rows = min(kRows, R - r0);

  pdl_wait();
  pdl_launch();
  const int first = a.seq_lens[b] - a.Lq;  // position of query token 0
  // (a length beyond the block table would be an error of the caller: no key past it is read)
  const int p_hi = min(first + Row(a, h, r0 + rows - 1).t, a.max_blocks * 16 - 1);
  const int p_lo = max(0, first + Row(a, h, r0).t);
  const Visible vis(p_lo, p_hi, a.window, a.sinks);
  const int per = (vis.n + a.splits - 1) / a.splits;
  const int u0 = split * per, u1 = min(vis.n, u0 + per);

  // A page's K and V loads are issued as soon as the registers of the page before are used up --
  // K's after its scores, V's after its share of O -- so they are in flight during the rest of
  // that page; page ids are fetched one page further ahead.
  const int32_t* bt = a.bt + (size_t)b * a.max_blocks;
  const size_t head_off = (size_t)h * a.head_stride;
  uint4 kf[2][KC], vf[4][VC];
  // keys of a page that some query of the tile sees: a hidden key is not loaded, so what its slot
  // holds does not matter
  auto seen = [&](int j) { return j <= p_hi && (j >= vis.lo || j < a.sinks); };
  // every key of the page visible to every query row
  auto inner = [&](int j0) { return j0 + 15 <= p_lo && (j0 > p_hi - a.window || j0 + 15 < a.sinks); };
  auto load_k = [&](int j0, int pid) {
    const uint16_t* kp = a.kc + (size_t)pid * a.page_stride + head_off + g * D + t * 8;
    const bool in = inner(j0), s0 = in || seen(j0 + g), s1 = in || seen(j0 + g + 8);
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      kf[0][i] = ldg16_if(kp + 32 * i, s0);
      kf[1][i] = ldg16_if(kp + 8 * D + 32 * i, s1);
    }
  };
  auto load_v = [&](int j0, int pid) {
    const uint16_t* vp = a.vc + (size_t)pid * a.page_stride + head_off + 2 * t * D + g * 8;
    const bool in = inner(j0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = (r & 1) + 8 * (r >> 1);
      const bool ok = in || seen(j0 + 2 * t + k);
#pragma unroll
      for (int c = 0; c < VC; ++c) vf[r][c] = ldg16_if(vp + k * D + 64 * c, ok);
    }
  };
  int u = u0 + warp;
  int pid = u < u1 ? bt[vis.page(u)] : 0, pid_next = u + kWinWarps < u1 ? bt[vis.page(u + kWinWarps)] : 0;
  if (u < u1) {
    load_k(vis.page(u) * 16, pid);
    load_v(vis.page(u) * 16, pid);
  }

  // Q tile, rows past the last one zero
  for (int i = threadIdx.x; i < kRows * (D / 8); i += kWinThreads) {
    const int r = i / (D / 8), c = i % (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const Row q(a, h, r0 + r);
      v = *reinterpret_cast<const uint4*>(a.q + (((size_t)b * a.Lq + q.t) * a.Hq + q.head) * D + c * 8);
    }
    *reinterpret_cast<uint4*>(qs + r * QS + c * 8) = v;
  }
  int pos[2];  // positions of this lane's columns 2 t + {0, 1}
  float m[2], l[2], o[MT][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    pos[e] = 2 * t + e < rows ? first + Row(a, h, r0 + 2 * t + e).t : -1;
    m[e] = -INFINITY;
    l[e] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[j][c] = 0.f;
  __syncthreads();
  uint4 qf[KC];  // Q^T fragments
#pragma unroll
  for (int i = 0; i < KC; ++i) qf[i] = *reinterpret_cast<const uint4*>(qs + g * QS + (4 * i + t) * 8);

  for (; u < u1; u += kWinWarps) {
    const int j0 = vis.page(u) * 16;
    const bool more = u + kWinWarps < u1, in = inner(j0);
    const int j0_next = more ? vis.page(u + kWinWarps) * 16 : 0;
    pid = pid_next;
    if (u + 2 * kWinWarps < u1) pid_next = bt[vis.page(u + 2 * kWinWarps)];
    // (key g, column 2t), (g, 2t+1), (g+8, 2t), (g+8, 2t+1); two chains of products
    float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      mma_bf16_16816(s, kf[0][i].x, kf[1][i].x, kf[0][i].y, kf[1][i].y, qf[i].x, qf[i].y);
      mma_bf16_16816(s2, kf[0][i].z, kf[1][i].z, kf[0][i].w, kf[1][i].w, qf[i].z, qf[i].w);
    }
    if (more) load_k(j0_next, pid);
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = (s[c] + s2[c]) * a.scale_log2;
    if (!in) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + g + 8 * (c >> 1), p = pos[c & 1];
        if (!(j <= p && (j > p - a.window || j < a.sinks))) s[c] = -INFINITY;
      }
    }
    float mx[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
    if (__any_sync(0xffffffffu, mx[0] > m[0] + kSlack || mx[1] > m[1] + kSlack)) {
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
        const float mn = fmaxf(m[e], mx[e]);
        alpha[e] = mn == -INFINITY ? 1.f : ex2(m[e] - mn);
        m[e] = mn;
        l[e] *= alpha[e];
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        o[j][0] *= alpha[0];
        o[j][1] *= alpha[1];
        o[j][2] *= alpha[0];
        o[j][3] *= alpha[1];
      }
    }
    const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
    s[0] = ex2(s[0] - b0);
    s[1] = ex2(s[1] - b1);
    s[2] = ex2(s[2] - b0);
    s[3] = ex2(s[3] - b1);
    l[0] += s[0] + s[2];
    l[1] += s[1] + s[3];
    uint32_t hi0, lo0, hi1, lo1;
    split_bf2(s[0], s[1], hi0, lo0);
    split_bf2(s[2], s[3], hi1, lo1);
    hi0 = transpose8x8(hi0);
    hi1 = transpose8x8(hi1);
    lo0 = transpose8x8(lo0);
    lo1 = transpose8x8(lo1);
    // O^T tile j: rows g and g + 8 are d = 8 g + j and, 128 wide, 64 + 8 g + j; 64 wide, 8 g + j + 4
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int c1 = VC - 1, e1 = VC == 2 ? j : j + 4;
      const uint32_t sel0 = (j & 1) ? 0x7632u : 0x5410u, sel1 = (e1 & 1) ? 0x7632u : 0x5410u;
      const uint32_t a0 = prmt(part4(vf[0][0], j >> 1), part4(vf[1][0], j >> 1), sel0);
      const uint32_t a1 = prmt(part4(vf[0][c1], e1 >> 1), part4(vf[1][c1], e1 >> 1), sel1);
      const uint32_t a2 = prmt(part4(vf[2][0], j >> 1), part4(vf[3][0], j >> 1), sel0);
      const uint32_t a3 = prmt(part4(vf[2][c1], e1 >> 1), part4(vf[3][c1], e1 >> 1), sel1);
      mma_bf16_16816(o[j], a0, a1, a2, a3, hi0, hi1);
      mma_bf16_16816(o[j], a0, a1, a2, a3, lo0, lo1);
    }
    if (more) load_v(j0_next, pid);
  }

  // ---- the warps' shares of the split, in shared memory ----
  // A lane holds, of each of its columns, 8 consecutive d (and 8 more 64 further on, 128 wide):
  // 16-byte stores, the two halves in an order that keeps a quarter warp's on distinct banks.
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
    const int r = 2 * t + e;
    if (g == 0) sm_ml[warp][r] = make_float2(m[e], l[e]);
    float* dst = sm_o + (warp * kRows + r) * OS + 8 * g;
    if (r < rows) {
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        // 128 wide: d = 64 c + 8 g + 0..7 in tiles 0..7; 64 wide: tiles 0..3, upper rows second
        const int f = 2 * c + e, f2 = VC == 2 ? f : e + 2, j2 = VC == 2 ? 4 : 0;
        const float4 v0 = make_float4(o[0][f], o[1][f], o[2][f], o[3][f]);
        const float4 v1 = make_float4(o[j2][f2], o[j2 + 1][f2], o[j2 + 2][f2], o[j2 + 3][f2]);
        *reinterpret_cast<float4*>(dst + 64 * c + 4 * (t & 1)) = (t & 1) ? v1 : v0;
        *reinterpret_cast<float4*>(dst + 64 * c + 4 * ((t & 1) ^ 1)) = (t & 1) ? v0 : v1;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < rows) {  // the warps' weights in the split's sum, and its maximum and norm
    const int r = threadIdx.x;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) M = fmaxf(M, sm_ml[w][r].x);
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) {
      const float f = M == -INFINITY ? 0.f : ex2(sm_ml[w][r].x - M);
      sm_f[w][r] = f;
      L = fmaf(f, sm_ml[w][r].y, L);
    }
    sm_ml[0][r] = make_float2(M, L);
  }
  __syncthreads();
  const int pair = (b * a.Hkv + h) * a.tiles + tile;
  // row r, d .. d + 3 of the output (f: 1 / norm)
  auto store = [&](int r, int d, float4 v, float f) {
    const Row q(a, h, r0 + r);
    // (a row without position may hold sums over other rows' keys)
    const uint2 w = first + q.t < 0 ? make_uint2(0, 0) : make_uint2(pack_bf2(v.x * f, v.y * f), pack_bf2(v.z * f, v.w * f));
    *reinterpret_cast<uint2*>(a.out + (((size_t)b * a.Lq + q.t) * a.Hq + q.head) * D + d) = w;
  };
  float* po = a.part + ((size_t)pair * a.splits + split) * kRows * D;
  float2* pml = a.part_ml + ((size_t)pair * a.splits + split) * kRows;
  for (int i = threadIdx.x; i < rows * (D / 4); i += kWinThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) {
      const float f = sm_f[w][r];
      const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * kRows + r) * OS + d);
      O.x = fmaf(f, v.x, O.x);
      O.y = fmaf(f, v.y, O.y);
      O.z = fmaf(f, v.z, O.z);
      O.w = fmaf(f, v.w, O.w);
    }
    if (a.splits == 1)
      store(r, d, O, sm_ml[0][r].y > 0.f ? 1.f / sm_ml[0][r].y : 0.f);
    else
      *reinterpret_cast<float4*>(po + r * D + d) = O;
  }
  if (a.splits == 1) return;
  if (threadIdx.x < rows) pml[threadIdx.x] = sm_ml[0][threadIdx.x];

  // ---- the last split to finish joins them, in the order of the splits ----
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) is_last = atomicAdd(a.counters + pair, 1) == a.splits - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  const float* part = a.part + (size_t)pair * a.splits * kRows * D;
  const float2* part_ml = a.part_ml + (size_t)pair * a.splits * kRows;
  float* weight = sm_o;  // [rows][splits]: the splits' weights over the whole norm
  for (int r = warp; r < rows; r += kWinWarps) {
    float2 v[kMaxSplits / 32];
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
      const int s = lane + 32 * i;
      v[i] = s < a.splits ? __ldcg(part_ml + (size_t)s * kRows + r) : make_float2(-INFINITY, 0.f);
      M = fmaxf(M, v[i].x);
    }
    M = warp_max(M);
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
      v[i].x = M == -INFINITY ? 0.f : ex2(v[i].x - M);
      L = fmaf(v[i].x, v[i].y, L);
    }
    L = warp_sum(L);
    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i)
      if (lane + 32 * i < a.splits) weight[r * a.splits + lane + 32 * i] = v[i].x * inv;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (D / 4); i += kWinThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
      const float f = weight[r * a.splits + s];
      const float4 v = __ldcg(reinterpret_cast<const float4*>(part + ((size_t)s * kRows + r) * D + d));
      O.x = fmaf(f, v.x, O.x);
      O.y = fmaf(f, v.y, O.y);
      O.z = fmaf(f, v.z, O.z);
      O.w = fmaf(f, v.w, O.w);
    }
    store(r, d, O, 1.f);
  }
  if (threadIdx.x == 0) a.counters[pair] = 0;
}

struct WinPlan {
  int tiles, splits;
};

// Splits of the visible pages.  A CTA's time is its pages (4 warps) plus about four pages' worth
// of start, merge and store; the splits that need the least over the waves of resident CTAs.
WinPlan plan_window(int B, int Lq, int Hq, int Hkv, int D, int max_seq_len, int window, int sinks) {
  WinPlan p;
  p.tiles = ((Hq / Hkv) * Lq + kRows - 1) / kRows;
  const int64_t keys = std::min<int64_t>(max_seq_len, (int64_t)window + sinks + Lq);
  const int64_t pages = std::min<int64_t>((max_seq_len + 15) / 16, (keys + 15) / 16 + 1);
  const int64_t pairs = (int64_t)B * Hkv * p.tiles, slots = 148 * (D == 64 ? kCtasPerSm64 : kCtasPerSm128);
  int64_t best = INT64_MAX;
  p.splits = 1;
  for (int s = 1; s <= std::min<int64_t>(kMaxSplits, (pages + kWinWarps - 1) / kWinWarps); ++s) {
    if (s > 1 && pairs > kWinCounterBytes / 4) break;
    const int64_t waves = (pairs * s + slots - 1) / slots;
    const int64_t cost = waves * ((pages + (int64_t)kWinWarps * s - 1) / (kWinWarps * s) + 4);
    if (cost < best) {
      best = cost;
      p.splits = s;
    }
  }
  return p;
}

size_t window_ws_bytes(const WinPlan& p, int B, int Hkv, int D) {
  if (p.splits == 1) return kWinCounterBytes;
  return kWinCounterBytes + (size_t)B * Hkv * p.tiles * p.splits * kRows * (D + 2) * sizeof(float);
}

bool window_shape_ok(int B, int Lq, int Hq, int Hkv, int D, int max_seq_len, int window, int sinks) {
  return B > 0 && Lq > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && (D == 64 || D == 128) && max_seq_len > 0 &&
         max_seq_len <= (1 << 30) && window > 0 && sinks >= 0 && (int64_t)Lq * Hq <= (1 << 30) && Hkv <= 65535 &&
         B <= 65535;
}

// Above 64 query rows per kv head the tcgen05 kernel (window_prefill.cu) takes over, as one does for
// higgs_paged_attention.  It walks a tile's keys in one CTA, this file's kernel shares them out but
// reads them once per 8 rows.  Both measured, us, 32 / 8 heads, D = 128, one sequence, 1024 / 4096 /
// 8192 visible keys: 17 tokens (68 rows) tcgen05 26 / 72 / 132, split 13 / 24 / 39; 64 tokens 28 / 71 /
// 129 and 29 / 72 / 125; 200 tokens 29 / 74 / 134 and 52 / 182 / 356.  16 sequences, 1024 keys: 17 tokens
// 29 and 77.  So for one sequence of 17 to 64 tokens the split kernel would be up to three times
// faster, for batches and longer chunks the tcgen05 kernel is.
bool window_on_tc(int Lq, int Hq, int Hkv) { return prefill_attn_tc_on() && (int64_t)(Hq / Hkv) * Lq > 64; }

}  // namespace
}  // namespace higgs

using namespace higgs;

extern "C" size_t higgs_window_attention_workspace_size(int B, int Lq, int Hq, int Hkv, int D, int max_seq_len,
                                                        int window, int sinks) {
  if (!window_shape_ok(B, Lq, Hq, Hkv, D, max_seq_len, window, sinks)) return 0;
  if (window_on_tc(Lq, Hq, Hkv)) return kWinCounterBytes;
  window = std::min(window, max_seq_len);
  sinks = std::min(sinks, max_seq_len);
  return window_ws_bytes(plan_window(B, Lq, Hq, Hkv, D, max_seq_len, window, sinks), B, Hkv, D);
}

extern "C" int higgs_window_attention(higgs_ctx* ctx, const void* q, int B, int Lq, int Hq, int Hkv, int D,
                                      const void* k_cache, const void* v_cache, int64_t page_stride,
                                      int64_t head_stride, const int32_t* block_table, int max_blocks,
                                      const int32_t* seq_lens, int max_seq_len, int window, int sinks, float scale,
                                      void* out, void* workspace, size_t workspace_bytes, void* stream) {
  HG_CHECK_ARG(ctx && q && k_cache && v_cache && block_table && seq_lens && out && workspace,
               "higgs_window_attention: null argument");
  HG_CHECK_ARG(D == 64 || D == 128, "higgs_window_attention: D must be 64 or 128");
  HG_CHECK_ARG(window > 0 && sinks >= 0, "higgs_window_attention: needs window >= 1 and sinks >= 0");
  HG_CHECK_ARG(window_shape_ok(B, Lq, Hq, Hkv, D, max_seq_len, window, sinks),
               "higgs_window_attention: bad batch / head shape");
  HG_CHECK_ARG((int64_t)max_blocks * HIGGS_PAGE_SIZE >= max_seq_len && max_blocks <= (1 << 26),
               "higgs_window_attention: block table too short (or beyond 2^26 pages)");
  HG_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) &
                15) == 0 &&
                   page_stride % 8 == 0 && head_stride % 8 == 0 && page_stride > 0 && head_stride > 0,
               "higgs_window_attention: tensors, workspace and (positive) strides must be 16-byte aligned");
  HG_CHECK_ARG(scale > 0.f && scale < INFINITY, "higgs_window_attention: scale must be positive and finite");
  // a window or sinks past the longest sequence are the whole sequence
  window = std::min(window, max_seq_len);
  sinks = std::min(sinks, max_seq_len);
  const bool tc = window_on_tc(Lq, Hq, Hkv);
  const WinPlan p = plan_window(B, Lq, Hq, Hkv, D, max_seq_len, window, sinks);
  HG_CHECK_ARG(tc ? (int64_t)B * Lq * Hq <= (1 << 30)
                  : (int64_t)Hkv * p.tiles <= 65535 && (int64_t)Lq * (Hq / Hkv) * (Hq / Hkv) < ((int64_t)1 << 32),
               "higgs_window_attention: too many query rows");
  const size_t need = tc ? kWinCounterBytes : window_ws_bytes(p, B, Hkv, D);
  if (workspace_bytes < need)
    return fail(HIGGS_ERR_WORKSPACE,
                "higgs_window_attention: workspace too small (need " + std::to_string(need) + " bytes)");
  HG_DEVICE(ctx);
  if (tc) {
    HG_CUDA(launch_window_prefill(q, B, Lq, Hq, Hkv, D, k_cache, v_cache, page_stride, head_stride, block_table,
                                  max_blocks, seq_lens, window, sinks, scale, out, (int*)workspace, tc_err_ptr(),
                                  (cudaStream_t)stream));
    return HIGGS_OK;
  }
  WinArgs a;
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  a.bt = block_table;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.Lq = Lq;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.inv_G = (uint32_t)((((uint64_t)1 << 32) + a.G - 1) / a.G);
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (uint16_t*)out;
  a.splits = p.splits;
  a.tiles = p.tiles;
  a.counters = (int*)workspace;
  a.part = (float*)((char*)workspace + kWinCounterBytes);
  a.part_ml = (float2*)(a.part + (size_t)B * Hkv * p.tiles * p.splits * kRows * D);
  cudaStream_t st = (cudaStream_t)stream;
  HG_CUDA(launch_pdl(D == 64 ? window_decode_kernel<64> : window_decode_kernel<128>,
                     dim3(p.splits, Hkv * p.tiles, B), dim3(kWinThreads), 0, st, a));
  return HIGGS_OK;
}
