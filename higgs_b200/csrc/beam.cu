// beam.cu -- beam search's selection: the n best continuations over the beams and the vocabulary
// of each request.  No reference counterpart (its generation loops are greedy or sampled,
// crates/higgs-models/src/lib.rs:373-385); the logits, their order (NaN last, the lower index on
// ties) and the log-probabilities are those of higgs_logprobs (lib.rs:495-533).
//
//   key(w, v) = score[w] + x[w, v] - log sum_u exp x[w, u]
//
// Within a beam the keys are ordered as the logits are, so one pass over a row gives all that is
// needed of it: the sum of its exponentials and its n largest logits.  A row is cut into rounds of
// 4096 logits, and the rounds of all rows into shares for as many CTAs as are resident at once; a
// CTA takes its share row by row, 16 logits per thread and round, the next round's in flight while
// it works on these.  Each warp writes the round's maximum and sum of exponentials, and collects
// the logits that reach a bound to which all eight warps contribute (scan_rounds): after the first
// rounds they are few, so the common logit costs a comparison and an exponential.  A warp that
// collects 32 sorts them (a bitonic network) and keeps the best, so no order of the logits needs
// more room; at the end the CTA's few candidates are ranked by counting those above each.
//
// The CTA that completes a request's last round joins its lists.  A row's exponentials and their sums
// are in f32 (a few ulps each; the log sum is held to 2^-20 by the tests), the logarithm, the key and
// its order in 64 bits: candidates of two beams closer than the log sums' error may change places,
// candidates of one beam or of equal rows never.  A histogram over the leading bits bounds the n-th
// best, and what reaches the bound is ranked as above.
//
// Keys are unique (value, then index), and the sums of a round depend on its logits alone and are
// added in the order of the rounds: equal rows give equal keys, and results do not depend on
// scheduling or on how the rounds are shared out.
//
// Bound: HBM, 4 bytes per logit of a beam that is alive.  B200: 32 requests x 16 beams x 151936
// logits, 32 best (311 MB) 73 us = 4.3 TB/s: nine CTAs in ten end their scans 48 to 62 us after the
// start (equal shares, unequal speeds), and the last one's list and join take 10 more; 8 x 8 beams,
// 16 best (39 MB) 19.7 us; one request 8.6 us, a chain of launch, one round, list, counter, log
// sums and join.  Where fewer than n lists of more than 2048 entries hold anything (the first step of
// wide beams), the join walks all entries: 32 us for 4 x 16 beams, 32 best; 64 us for 1 x 32.
#include <algorithm>

#include "common.cuh"

namespace higgs {
namespace {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamElems = 16;                         // logits per lane and round
constexpr int kBeamRound = kBeamThreads * kBeamElems;  // logits per CTA and round
constexpr int kMaxOut = 32;                            // n_out: one key per lane of a warp
constexpr int kMaxBeams = 32;
constexpr int kMaxBeamVocab = 163840;
constexpr int kUnitsPerLane = (kMaxBeamVocab + kBeamRound - 1) / kBeamRound * kBeamWarps / 32;  // sums of a row
constexpr int kBeamCounterBytes = 4096;
constexpr float kLowest = -3.402823466e38f;  // of the finite values
constexpr int kBeamCtasPerSm = 3;  // resident at once (registers)

struct BeamArgs {
  const float* logits;
  const float* scores;
  int B, beams, V, n;
  // rounds of a row; places of a row in the order of all rounds (`rounds`, or more to make shares
  // end with the rows); places of a CTA; CTAs that may share a row
  int rounds, stride, share, lists;
  uint32_t inv_n;            // 2^32 / n, rounded up
  int* counters;             // [B] places done, zero before the launch and after it
  float2* sums;              // [B * beams][rounds][warps] maximum, sum of exp(x - maximum)
  unsigned long long* tops;  // [B * beams][lists][n] argmax keys, largest first, 0 = none
  float* out_scores;
  int32_t* out_beams;
  int32_t* out_tokens;
};

// A logit of a row: the key orders by value, then by lower index; 0 is "none".
struct LogitKey {
  unsigned long long k;
  __device__ static LogitKey none() { return {0ull}; }
  __device__ bool over(const LogitKey& o) const { return k > o.k; }
  __device__ bool is_none() const { return k == 0; }
  __device__ LogitKey shfl_xor(int m) const { return {__shfl_xor_sync(0xffffffffu, k, m)}; }
  __device__ LogitKey from(int lane) const { return {__shfl_sync(0xffffffffu, k, lane)}; }
};

// A candidate of a request: its score in 64 bits, as an integer of the same order (64-bit
// floating-point comparisons are slow), then the lower beam * V + token.
struct BeamKey {
  unsigned long long s;
  uint32_t at;
  __device__ static BeamKey none() { return {0ull, 0xffffffffu}; }
  __device__ static BeamKey of(double score, uint32_t at) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(score + 0.0);  // -0 is +0
    return {(u >> 63) ? ~u : u | (1ull << 63), at};
  }
  __device__ double score() const {
    return __longlong_as_double((long long)((s >> 63) ? s & ~(1ull << 63) : ~s));
  }
  __device__ bool over(const BeamKey& o) const { return s > o.s || (s == o.s && at < o.at); }
  __device__ bool is_none() const { return s == 0; }
  __device__ uint32_t high() const { return (uint32_t)(s >> 32); }  // ordered as the keys are, with ties
  __device__ BeamKey shfl_xor(int m) const {
    return {__shfl_xor_sync(0xffffffffu, s, m), __shfl_xor_sync(0xffffffffu, at, m)};
  }
  __device__ BeamKey from(int lane) const {
    return {__shfl_sync(0xffffffffu, s, lane), __shfl_sync(0xffffffffu, at, lane)};
  }
};

__device__ __forceinline__ float logit_of(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int index_of(unsigned long long k) { return (int)(0xffffffffu - (uint32_t)k); }

// lane i of the warp gets the i-th largest of its 32 keys (bitonic network; it runs rarely, so its
// loops stay loops)
template <typename Key>
__device__ __forceinline__ Key warp_sort(Key k) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll 1
    for (int d = size >> 1; d > 0; d >>= 1) {
      const Key o = k.shfl_xor(d);
      const bool keep_larger = ((lane & size) == 0) == ((lane & d) == 0);
      if (o.over(k) == keep_larger) k = o;
    }
  return k;
}

// the 32 largest of two lists sorted largest first, sorted: the larger of a[i] and b[31 - i] are
// those 32, and bitonic
template <typename Key>
__device__ __forceinline__ Key warp_merge(Key a, Key b_rev) {
  Key k = b_rev.over(a) ? b_rev : a;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int d = 16; d > 0; d >>= 1) {
    const Key o = k.shfl_xor(d);
    if (o.over(k) == ((lane & d) == 0)) k = o;
  }
  return k;
}

// The keys a warp has been given: fewer than 32 pending ones, and the 32 best of those before,
// sorted, one per lane; `edge` is the n-th of these.
template <typename Key>
struct WarpTop {
  Key best, edge;
  Key* pending;  // [64] of this warp
  int n_pending, n;
  __device__ WarpTop(Key* buf, int n_) : best(Key::none()), edge(Key::none()), pending(buf), n_pending(0), n(n_) {}
  // called by the whole warp: adds k of the lanes with `add`
  __device__ void push(bool add, Key k) {
    const uint32_t lanes = __ballot_sync(0xffffffffu, add);
    if (!lanes) return;
    if (add) pending[n_pending + __popc(lanes & ((1u << (threadIdx.x & 31)) - 1))] = k;
    n_pending += __popc(lanes);
    __syncwarp();
    if (n_pending >= 32) {
      const int lane = threadIdx.x & 31;
      k = warp_sort(pending[lane]);
      const Key rest = pending[32 + lane];
      __syncwarp();
      pending[lane] = rest;
      n_pending -= 32;
      __syncwarp();
      best = warp_merge(best, k.from(31 - lane));
      edge = best.from(n - 1);
    }
  }
};

constexpr int kMaxCand = kBeamWarps * 64;
constexpr int kMaxLists = 512;    // of a request
constexpr int kMaxDirect = 2048;  // entries of lists that are joined directly
static_assert(kBeamCtasPerSm * 148 + 2 * kMaxBeams <= kMaxLists, "shares that a request's rows can meet");
template <typename Key>
struct TopShared {
  Key pending[kBeamWarps][64];
  Key cand[kMaxCand];
  int n_cand;
};
struct BoundShared {
  int bins[kBeamThreads];
  int warp_count[kBeamWarps];
  uint32_t lo, hi;
  int pick, above, reach, total;
};

struct JoinShared {
  TopShared<BeamKey> top;
  float2 total[kMaxBeams];         // log sums: maximum, sum
  double beam_offset[kMaxBeams];   // score - log sum, NaN: no candidates
  double offset[kMaxLists];        // of the list's beam
  uint32_t base[kMaxLists];        // beam * V
  uint32_t high[kMaxDirect];
  BoundShared bound;
};
union BeamShared {
  __device__ BeamShared() {}
  TopShared<LogitKey> row;
  JoinShared join;
};

// A bound that n or more (and mostly few more) of the m values reach, or 1, which bounds nothing, if
// there are fewer than n: the least of them is no bound for what the values are the heads of.  Zeros
// do not count.  Each pass spreads the range that holds the n-th value over 256 bins.
__device__ __forceinline__ uint32_t block_bound(const uint32_t* v, int m, int n, BoundShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    sh.lo = 0xffffffffu;
    sh.hi = 0;
  }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = threadIdx.x; i < m; i += kBeamThreads)
    if (v[i]) {
      lo = min(lo, v[i]);
      hi = max(hi, v[i]);
    }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0 && hi) {
    atomicMin(&sh.lo, lo);
    atomicMax(&sh.hi, hi);
  }
  __syncthreads();
  lo = sh.lo;
  hi = sh.hi;
  if (hi == 0) return 1;
  while (true) {
    const uint32_t range = hi - lo;
    const int shift = max(0, 24 - __clz(range));  // (range >> shift) < 256
    sh.bins[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kBeamThreads)
      if (v[i] >= lo && v[i] <= hi) atomicAdd(&sh.bins[(v[i] - lo) >> shift], 1);
    __syncthreads();
    const int own = sh.bins[threadIdx.x];
    int c = own;  // values in this bin and the ones above it
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_down_sync(0xffffffffu, c, d);
      if (lane + d < 32) c += x;
    }
    if (lane == 0) sh.warp_count[warp] = c;
    __syncthreads();
#pragma unroll
    for (int w = 1; w < kBeamWarps; ++w)
      if (w > warp) c += sh.warp_count[w];
    if (c >= n && c - own < n) {
      sh.pick = threadIdx.x;
      sh.above = c - own;
      sh.reach = c;
    }
    if (threadIdx.x == 0) sh.total = c;
    __syncthreads();
    if (sh.total < n) return 1;  // (in the first pass: later ones hold the n-th)
    lo += (uint32_t)sh.pick << shift;
    if (shift == 0 || sh.reach <= n + 8) return lo;
    hi = min(hi, lo + (1u << shift) - 1);
    n -= sh.above;
  }
}

// put(rank, key) for the n best of the candidates, each ranked by counting those over it
template <typename Key, typename Put>
__device__ __forceinline__ void rank_all(const Key* cand, int count, int n, Put put) {
  for (int i = threadIdx.x; i < count; i += kBeamThreads) {
    const Key k = cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) rank += cand[j].over(k);
    if (rank < n) put(rank, k);
  }
}

// put(rank, key) for the n best keys that the CTA's warps hold, of those for which keep(key); what
// is returned is n or more, or the count of keys if those are fewer.
template <typename Key, typename Keep, typename Put>
__device__ __forceinline__ int rank_tops(const WarpTop<Key>& top, TopShared<Key>& sh, int n, Keep keep, Put put) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) sh.n_cand = 0;
  __syncthreads();
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const Key k = half ? (lane < top.n_pending ? top.pending[lane] : Key::none()) : top.best;
    const bool add = !k.is_none() && keep(k);
    const uint32_t lanes = __ballot_sync(0xffffffffu, add);
    int at = 0;
    if (lane == 0 && lanes) at = atomicAdd(&sh.n_cand, __popc(lanes));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(lanes & ((1u << lane) - 1));
    if (add) sh.cand[at] = k;
  }
  __syncthreads();
  rank_all(sh.cand, sh.n_cand, n, put);
  return sh.n_cand;
}

// largest of the warp's values
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// the part-th largest of the lanes' values
__device__ __forceinline__ float warp_nth(float v, int part) {
  for (int i = 1; i < part; ++i) {
    const uint32_t top_lanes = __ballot_sync(0xffffffffu, v == redux_max(v));
    if ((int)(threadIdx.x & 31) == __ffs(top_lanes) - 1) v = -INFINITY;
  }
  return redux_max(v);
}

// The least of the warps' shares: if each is no larger than `part` values of its warp, where 8
// parts are n or more, a value below it is not among the n largest.
__device__ __forceinline__ float least_share(const volatile float* shares) {
  float least = shares[0];
#pragma unroll
  for (int i = 1; i < kBeamWarps; ++i) least = fminf(least, shares[i]);
  return least;
}

// A thread's logits of a round: VEC: 16-byte loads, four consecutive each; else one by one.  (Rows
// of one launch are all loaded the same way, so equal rows still give equal sums.)
template <bool VEC>
__device__ __forceinline__ int elem(int e) {
  return VEC ? 4 * kBeamThreads * (e >> 2) + (e & 3) : kBeamThreads * e;
}
template <bool VEC>
__device__ __forceinline__ void load_round(float (&d)[kBeamElems], const float* x, int at, int end) {
  const float* p = x + at;
  const int left = end - at;  // (a multiple of 4 for 16-byte loads)
  constexpr int step = VEC ? 4 : 1;
  if (elem<VEC>(kBeamElems - step) < left) {
#pragma unroll
    for (int e = 0; e < kBeamElems; e += step) {
      if (VEC) {
        const float4 q = __ldcs(reinterpret_cast<const float4*>(p + elem<VEC>(e)));
        d[e] = q.x, d[e + 1] = q.y, d[e + 2] = q.z, d[e + 3] = q.w;
      } else {
        d[e] = __ldcs(p + elem<VEC>(e));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kBeamElems; ++e) d[e] = elem<VEC>(e) < left ? __ldcs(p + elem<VEC>(e)) : -INFINITY;
  }
}

// sum of exp(v - m), two values to an instruction
__device__ __forceinline__ float exp_sum(const float (&v)[kBeamElems], float m) {
  const float2 neg_m = make_float2(-m, -m), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int e = 0; e < kBeamElems; e += 2) {
    const float2 t = __fmul2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), neg_m), log2e);
    float2 p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p.y) : "f"(t.y));
    sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], p);
  }
  sum[0] = __fadd2_rn(sum[0], sum[1]);
  return sum[0].x + sum[0].y;
}

// v[pick]
__device__ __forceinline__ float pick_elem(const float (&v)[kBeamElems], int pick) {
  float t[kBeamElems];
#pragma unroll
  for (int e = 0; e < kBeamElems; ++e) t[e] = v[e];
#pragma unroll
  for (int w = kBeamElems / 2; w > 0; w >>= 1)
#pragma unroll
    for (int e = 0; e < w; ++e) t[e] = (pick & w) ? t[e + w] : t[e];
  return t[0];
}

// Rounds [r0, r1) of a row: their sums, and their n largest logits to list[0 .. n), largest first.
template <bool VEC>
__device__ __forceinline__ void scan_rounds(const BeamArgs& a, int row, int r0, int r1, unsigned long long* list,
                                            TopShared<LogitKey>& sh, volatile float* shares) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* x = a.logits + (size_t)row * a.V;
  float2* sums = a.sums + ((size_t)row * a.rounds + r0) * kBeamWarps + warp;
  const int end = min(a.V, r1 * kBeamRound);
  int at = r0 * kBeamRound + threadIdx.x * (VEC ? 4 : 1);
  WarpTop<LogitKey> top(sh.pending[warp], a.n);
  // Shares are of the lanes' maxima so far.  They only rise, so one read late is a bound still;
  // the first round waits for all of them.
  const int part = (a.n + kBeamWarps - 1) / kBeamWarps;
  float lane_max = -INFINITY, share = -INFINITY, edge = kLowest;
  float v[kBeamElems], next[kBeamElems];
  load_round<VEC>(next, x, at, end);
  for (int r = r0; r < r1; ++r, at += kBeamRound, sums += kBeamWarps) {
    float mx = -INFINITY;  // (fmaxf passes a NaN by)
#pragma unroll
    for (int e = 0; e < kBeamElems; ++e) {
      v[e] = next[e];
      mx = fmaxf(mx, v[e]);
    }
    if (r + 1 < r1) load_round<VEC>(next, x, at + kBeamRound, end);
    const float m = redux_max(mx), mm = m == -INFINITY ? 0.f : m;
    if (m > share || r == r0) {
      lane_max = fmaxf(lane_max, mx);
      share = warp_nth(lane_max, part);
      if (lane == 0) shares[warp] = share;
      if (r == r0) __syncthreads();
    }
    float s = warp_sum(exp_sum(v, mm));
    if (s != s) {  // a NaN logit has no mass
#pragma unroll
      for (int e = 0; e < kBeamElems; ++e) v[e] = fmaxf(v[e], -INFINITY);
      s = warp_sum(exp_sum(v, mm));
    }
    if (lane == 0) *sums = make_float2(m, s);
    edge = fmaxf(edge, least_share(shares));
    if (m >= edge) {
      uint32_t over = 0;
#pragma unroll
      for (int e = 0; e < kBeamElems; ++e) over |= (uint32_t)(v[e] >= edge) << e;
      while (__any_sync(0xffffffffu, over != 0)) {  // one of each lane at a time
        const int pick = __ffs(over) - 1;
        const LogitKey k{argmax_key(pick_elem(v, pick), at + elem<VEC>(pick))};
        top.push(over != 0 && k.over(top.edge), k);
        over &= over - 1;
      }
      if (!top.edge.is_none()) edge = fmaxf(edge, logit_of(top.edge.k));
    }
  }
  __threadfence();  // the sums, before the rounds are counted
  __syncthreads();
  edge = fmaxf(kLowest, least_share(shares));
  const int count = rank_tops(
      top, sh, a.n, [&](LogitKey k) { return logit_of(k.k) >= edge; }, [&](int r, LogitKey k) { list[r] = k.k; });
  for (int r = count + threadIdx.x; r < a.n; r += kBeamThreads) list[r] = 0;
}

// The n best of request b from its rows' sums and lists.
__device__ __forceinline__ void join_request(const BeamArgs& a, int b, JoinShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // A beam's lists are those of the CTAs whose shares meet its row.
  const int lists = a.beams * a.lists, entries = lists * a.n;
  const unsigned long long* tops = a.tops + (size_t)b * entries;
  const bool direct = entries <= kMaxDirect;
  unsigned long long raw[kMaxDirect / kBeamThreads];
  if (direct) {
#pragma unroll
    for (int e = 0; e < kMaxDirect / kBeamThreads; ++e) {
      const int i = threadIdx.x + e * kBeamThreads;
      raw[e] = i < entries ? __ldcg(tops + i) : 0;
    }
  }
  // log sums: a warp adds up a row's rounds, then a lane takes each row's logarithm
  const int units = a.rounds * kBeamWarps;
  for (int w = warp; w < a.beams; w += kBeamWarps) {
    const int row = b * a.beams + w;
    float m = -INFINITY, z = 0.f;
    if (isfinite(a.scores[row])) {
      const float2* p = a.sums + (size_t)row * units;
      float2 q[kUnitsPerLane];
#pragma unroll
      for (int i = 0; i < kUnitsPerLane; ++i) {
        q[i] = lane + 32 * i < units ? __ldcg(p + lane + 32 * i) : make_float2(-INFINITY, 0.f);
        m = fmaxf(m, q[i].x);
      }
      m = redux_max(m);
#pragma unroll
      for (int i = 0; i < kUnitsPerLane; ++i)
        if (q[i].x != -INFINITY) z = fmaf(q[i].y, __expf(q[i].x - m), z);
      z = warp_sum(z);
    }
    if (lane == 0) sh.total[w] = make_float2(m, z);
  }
  __syncthreads();
  if (threadIdx.x < a.beams) {
    // score - log sum; NaN marks a beam that gives no candidates
    const float2 t = sh.total[threadIdx.x];
    sh.beam_offset[threadIdx.x] =
        isfinite(t.x) ? (double)a.scores[b * a.beams + threadIdx.x] - ((double)t.x + log((double)t.y)) : NAN;
  }
  __syncthreads();
  for (int l = threadIdx.x; l < lists; l += kBeamThreads) {
    const int w = l / a.lists, row = b * a.beams + w;
    const int n_lists = ((row + 1) * a.stride - 1) / a.share - row * a.stride / a.share + 1;
    sh.offset[l] = l - w * a.lists < n_lists ? sh.beam_offset[w] : NAN;
    sh.base[l] = (uint32_t)(w * a.V);
  }
  __syncthreads();
  auto key_of = [&](int i, unsigned long long k) {
    const int list = a.n == 1 ? i : (int)__umulhi((uint32_t)i, a.inv_n);
    const double off = sh.offset[list];
    return off == off && k != 0 ? BeamKey::of(off + (double)logit_of(k), sh.base[list] + index_of(k)) : BeamKey::none();
  };
  auto put = [&](int r, BeamKey k) {
    const size_t o = (size_t)b * a.n + r;
    const uint32_t w = k.at / (uint32_t)a.V;
    a.out_scores[o] = (float)k.score();
    a.out_beams[o] = (int32_t)w;
    a.out_tokens[o] = (int32_t)(k.at - w * a.V);
  };
  // Few entries: a bound that hardly more than n of them reach, and a rank for each of those.  Many
  // (so many lists), or too many of one value: entries no better than the n-th of the lists' heads
  // are left out -- none where fewer than n lists have one: dead beams and masked places have no
  // list -- and the warps sort the rest.
  int count = kMaxCand + 1;
  if (direct) {
    BeamKey key[kMaxDirect / kBeamThreads];
#pragma unroll
    for (int e = 0; e < kMaxDirect / kBeamThreads; ++e) {
      const int i = threadIdx.x + e * kBeamThreads;
      key[e] = raw[e] ? key_of(i, raw[e]) : BeamKey::none();
      if (i < entries) sh.high[i] = key[e].high();
    }
    if (threadIdx.x == 0) sh.top.n_cand = 0;
    const uint32_t bound = block_bound(sh.high, entries, a.n, sh.bound);
#pragma unroll
    for (int e = 0; e < kMaxDirect / kBeamThreads; ++e)
      if (key[e].high() >= bound) {
        const int at = atomicAdd(&sh.top.n_cand, 1);
        if (at < kMaxCand) sh.top.cand[at] = key[e];
      }
    __syncthreads();
    count = sh.top.n_cand;
    if (count <= kMaxCand) rank_all(sh.top.cand, count, a.n, put);
  }
  if (count > kMaxCand) {
    __syncthreads();
    for (int l = threadIdx.x; l < lists; l += kBeamThreads) sh.high[l] = key_of(l * a.n, __ldcg(tops + l * a.n)).high();
    const uint32_t bound = block_bound(sh.high, lists, a.n, sh.bound);
    WarpTop<BeamKey> top(sh.top.pending[warp], a.n);
    for (int i0 = warp * 32; i0 < entries; i0 += kBeamThreads) {
      const int i = i0 + lane;
      const BeamKey k = i < entries ? key_of(i, __ldcg(tops + i)) : BeamKey::none();
      top.push(k.high() >= bound && k.over(top.edge), k);
    }
    count = rank_tops(top, sh.top, a.n, [](BeamKey) { return true; }, put);
  }
  for (int r = count + threadIdx.x; r < a.n; r += kBeamThreads) {
    const size_t o = (size_t)b * a.n + r;
    a.out_scores[o] = -INFINITY;
    a.out_beams[o] = -1;
    a.out_tokens[o] = -1;
  }
  if (threadIdx.x == 0) a.counters[b] = 0;
}

template <bool VEC>
__global__ void __launch_bounds__(kBeamThreads, kBeamCtasPerSm) beam_select_kernel(BeamArgs a) {
  __shared__ BeamShared sh;
  __shared__ volatile float shares[kBeamWarps];
  __shared__ int is_last;
  pdl_wait();
  pdl_launch();
  const int g_end = min((int)(blockIdx.x + 1) * a.share, a.B * a.beams * a.stride);
  for (int g = blockIdx.x * a.share; g < g_end;) {
    const int row = g / a.stride, r0 = g - row * a.stride, r1 = min(a.stride, r0 + g_end - g), b = row / a.beams;
    if (r0 < a.rounds && isfinite(a.scores[row])) {  // a dead beam's logits are not read
      const int list = blockIdx.x - row * a.stride / a.share;
      scan_rounds<VEC>(a, row, r0, min(r1, a.rounds), a.tops + ((size_t)row * a.lists + list) * a.n, sh.row, shares);
      __threadfence();
      __syncthreads();
    }
    if (threadIdx.x == 0) is_last = atomicAdd(a.counters + b, r1 - r0) + r1 - r0 == a.beams * a.stride;
    __syncthreads();
    if (is_last) {
      __threadfence();
      join_request(a, b, sh.join);
    }
    __syncthreads();
    g += r1 - r0;
  }
}

bool beam_shape_ok(int B, int beams, int V, int n_out) {
  return B > 0 && B <= kBeamCounterBytes / 4 && beams > 0 && beams <= kMaxBeams && V > 0 && V <= kMaxBeamVocab &&
         n_out > 0 && n_out <= kMaxOut;
}

// Shares of all rows' rounds for the CTAs that are resident at once: either equal ones, which may
// run on from one row into the next -- a second start and list, about three rounds' time (measured)
// -- or equal parts of each row.
struct BeamPlan {
  int rounds, stride, share, lists, ctas;
};
BeamPlan plan_beam(int B, int beams, int V) {
  BeamPlan p;
  const int rows = B * beams, slots = kBeamCtasPerSm * 148;
  p.rounds = p.stride = (V + kBeamRound - 1) / kBeamRound;
  p.share = (rows * p.rounds + slots - 1) / slots;
  p.lists = (p.rounds + p.share - 2) / p.share + 1;
  if (rows <= slots) {
    const int share = (p.rounds + slots / rows - 1) / (slots / rows);
    if (share <= p.share + 3) {
      p.share = share;
      p.lists = (p.rounds + share - 1) / share;
      p.stride = p.lists * share;
    }
  }
  p.ctas = (rows * p.stride + p.share - 1) / p.share;
  return p;
}

size_t beam_ws_bytes(int B, int beams, int V, int n_out) {
  const BeamPlan p = plan_beam(B, beams, V);
  return kBeamCounterBytes + (size_t)B * beams *
                                 (p.rounds * kBeamWarps * sizeof(float2) + p.lists * n_out * sizeof(unsigned long long));
}

}  // namespace
}  // namespace higgs

using namespace higgs;

extern "C" size_t higgs_beam_select_workspace_size(int B, int beams, int V, int n_out) {
  return beam_shape_ok(B, beams, V, n_out) ? beam_ws_bytes(B, beams, V, n_out) : 0;
}

extern "C" int higgs_beam_select(higgs_ctx* ctx, const float* logits, const float* scores, int B, int beams, int V,
                                 int n_out, float* out_scores, int32_t* out_beams, int32_t* out_tokens,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  HG_CHECK_ARG(beam_shape_ok(B, beams, V, n_out),
               "higgs_beam_select: B 1..1024, beams 1..32, V 1..163840, n_out 1..32");
  HG_CHECK_ARG(ctx && logits && scores && out_scores && out_beams && out_tokens && workspace,
               "higgs_beam_select: null argument");
  HG_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "higgs_beam_select: workspace must be 16-byte aligned");
  const size_t need = beam_ws_bytes(B, beams, V, n_out);
  if (workspace_bytes < need)
    return fail(HIGGS_ERR_WORKSPACE,
                "higgs_beam_select: workspace too small (need " + std::to_string(need) + " bytes)");
  HG_DEVICE(ctx);
  BeamArgs a;
  a.logits = logits;
  a.scores = scores;
  a.B = B;
  a.beams = beams;
  a.V = V;
  a.n = n_out;
  const BeamPlan p = plan_beam(B, beams, V);
  a.rounds = p.rounds;
  a.stride = p.stride;
  a.share = p.share;
  a.lists = p.lists;
  a.inv_n = (uint32_t)((((uint64_t)1 << 32) + n_out - 1) / n_out);
  a.counters = (int*)workspace;
  a.sums = (float2*)((char*)workspace + kBeamCounterBytes);
  a.tops = (unsigned long long*)(a.sums + (size_t)B * beams * p.rounds * kBeamWarps);
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  // 16-byte loads where every row starts on a 16-byte boundary
  const bool vec = V % 4 == 0 && ((uintptr_t)logits & 15) == 0;
  HG_CUDA(launch_pdl(vec ? beam_select_kernel<true> : beam_select_kernel<false>, dim3(p.ctas), dim3(kBeamThreads), 0,
                     (cudaStream_t)stream, a));
  return HIGGS_OK;
}
