// beam.cu -- beam search's selection: the n best continuations over the beams and the vocabulary
// of each request.  No reference counterpart (its generation loops are greedy or sampled,
// crates/higgs-models/src/lib.rs:373-385); the logits, their order (NaN last, the lower index on
// ties) and the log-probabilities are those of higgs_logprobs (lib.rs:495-533).
//
//   key(w, v) = score[w] + x[w, v] - log sum_u exp x[w, u]
//
// Within a beam the keys are ordered as the logits are, so one pass over a row gives all that is
// needed of it: the sum of its exponentials and its n largest logits.  A CTA takes a chunk of a
// row into registers, once: the chunk's maximum and its sum of exponentials relative to it, and
// the chunk's n largest logits -- the n-th largest of the threads' own maxima is a lower bound of
// the chunk's n-th largest, so the few logits above it are gathered and ranked.  The last CTA of a
// request to finish joins the chunks: log sums, then the n best of score - log sum + logit, in 64
// bits (which of two near candidates wins is decided by the difference of two such sums), found
// by the same bound over the heads of the sorted lists.
//
// Keys are unique (value, then index), so the gathered lists are bounded whatever the data; sums
// run in an order fixed by the chunk's index alone, so equal rows give equal keys and results do
// not depend on scheduling.  Bound: HBM, 4 bytes per logit of a beam that is alive.
#include <algorithm>

#include "common.cuh"

namespace higgs {
namespace {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamElems = 32;                           // logits per thread
constexpr int kBeamChunk = kBeamThreads * kBeamElems;    // logits per CTA
constexpr int kMaxOut = 32;                              // n_out: one warp sorts that many keys
constexpr int kMaxBeams = 32;
constexpr int kMaxBeamVocab = 163840;
constexpr int kMaxChunks = (kMaxBeamVocab + kBeamChunk - 1) / kBeamChunk;
constexpr int kListsPerThread = (kMaxBeams * kMaxChunks + kBeamThreads - 1) / kBeamThreads;
constexpr int kBeamCounterBytes = 4096;

struct BeamArgs {
  const float* logits;
  const float* scores;
  int beams, V, n, chunks;
  int* counters;             // [B] chunks done, zero before the launch and after it
  float2* sums;              // [B * beams][chunks] maximum, sum of exp(x - maximum)
  unsigned long long* tops;  // [B * beams][chunks][n] argmax keys, largest first, 0 = none
  float* out_scores;
  int32_t* out_beams;
  int32_t* out_tokens;
};

// A logit of a chunk: the key orders by value, then by lower index; 0 is "none".
struct LogitKey {
  unsigned long long k;
  __device__ static LogitKey none() { return {0ull}; }
  __device__ bool over(const LogitKey& o) const { return k > o.k; }
  __device__ bool is_none() const { return k == 0; }
  __device__ LogitKey shfl_xor(int m) const { return {__shfl_xor_sync(0xffffffffu, k, m)}; }
};

// A candidate of a request: its score in 64 bits, then the lower beam * V + token.
struct BeamKey {
  double s;
  uint32_t at;
  __device__ static BeamKey none() { return {-INFINITY, 0xffffffffu}; }
  __device__ bool over(const BeamKey& o) const { return s > o.s || (s == o.s && at < o.at); }
  __device__ bool is_none() const { return at == 0xffffffffu; }
  __device__ BeamKey shfl_xor(int m) const {
    return {__shfl_xor_sync(0xffffffffu, s, m), __shfl_xor_sync(0xffffffffu, at, m)};
  }
};

__device__ __forceinline__ float logit_of(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int index_of(unsigned long long k) { return (int)(0xffffffffu - (uint32_t)k); }

// lane i of the warp gets the i-th largest of its 32 keys (bitonic network)
template <typename Key>
__device__ __forceinline__ Key warp_sort(Key k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
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
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const Key o = k.shfl_xor(d);
    if (o.over(k) == ((lane & d) == 0)) k = o;
  }
  return k;
}

// The n-th largest (n <= 32) of one key per thread, or `none` if fewer are given.
template <typename Key>
__device__ Key block_nth(Key k, int n, Key (*lists)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  k = warp_sort(k);
  for (int half = kBeamWarps / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) lists[warp - half][lane] = k;
    __syncthreads();
    if (warp < half) k = warp_merge(k, lists[warp][31 - lane]);
    __syncthreads();
  }
  if (warp == 0) lists[0][lane] = k;
  __syncthreads();
  return lists[0][n - 1];
}

struct ChunkShared {
  LogitKey lists[kBeamWarps / 2][32];
  LogitKey cand[kMaxOut * kBeamElems];  // at most n threads own a key over the bound
};
struct JoinShared {
  BeamKey lists[kBeamWarps / 2][32];
  BeamKey cand[kMaxOut * kListsPerThread * kMaxOut];
};
union BeamShared {
  ChunkShared c;
  JoinShared j;
};

// `cand` holds the n_cand keys that may be among the n largest: calls put(rank, key) for those.
template <typename Key, typename Put>
__device__ __forceinline__ void rank_candidates(const Key* cand, int n_cand, int n, Put put) {
  for (int i = threadIdx.x; i < n_cand; i += kBeamThreads) {
    const Key k = cand[i];
    int rank = 0;
    for (int j = 0; j < n_cand; ++j) rank += cand[j].over(k);
    if (rank < n) put(rank, k);
  }
}

__global__ void __launch_bounds__(kBeamThreads) beam_select_kernel(BeamArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  BeamShared& sh = *reinterpret_cast<BeamShared*>(smem_raw);
  __shared__ float warp_red[kBeamWarps];
  __shared__ int n_cand, is_last;
  __shared__ double offset[kMaxBeams];
  const int chunk = blockIdx.x, w = blockIdx.y, b = blockIdx.z;
  const int row = b * a.beams + w;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_wait();
  pdl_launch();
  const bool alive = isfinite(a.scores[row]);  // a dead beam's logits are not read
  if (alive) {
    const float* x = a.logits + (size_t)row * a.V;
    const int i0 = chunk * kBeamChunk + threadIdx.x;
    float v[kBeamElems];
#pragma unroll
    for (int e = 0; e < kBeamElems; ++e) {
      const int i = i0 + e * kBeamThreads;
      v[e] = i < a.V ? __ldcs(x + i) : -INFINITY;
    }
    float best = -INFINITY;
    int best_i = i0;
#pragma unroll
    for (int e = 0; e < kBeamElems; ++e) {
      v[e] = v[e] == v[e] ? v[e] : -INFINITY;  // NaN: no mass, never chosen
      if (v[e] > best) {
        best = v[e];
        best_i = i0 + e * kBeamThreads;
      }
    }
    float m = warp_max(best);
    if (lane == 0) warp_red[warp] = m;
    if (threadIdx.x == 0) n_cand = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBeamWarps; ++i) m = fmaxf(m, warp_red[i]);
    __syncthreads();
    const float mm = m == -INFINITY ? 0.f : m;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < kBeamElems; ++e) sum[e & 3] += __expf(v[e] - mm);
    const float s = warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (lane == 0) warp_red[warp] = s;

    const LogitKey mine = best == -INFINITY ? LogitKey::none() : LogitKey{argmax_key(best, best_i)};
    const LogitKey edge = block_nth(mine, a.n, sh.c.lists);
    if (!mine.is_none() && !edge.over(mine)) {
#pragma unroll
      for (int e = 0; e < kBeamElems; ++e) {
        const LogitKey k{argmax_key(v[e], i0 + e * kBeamThreads)};
        if (v[e] != -INFINITY && !edge.over(k)) sh.c.cand[atomicAdd(&n_cand, 1)] = k;
      }
    }
    __syncthreads();
    const int nc = n_cand;
    unsigned long long* top = a.tops + ((size_t)row * a.chunks + chunk) * a.n;
    rank_candidates(sh.c.cand, nc, a.n, [&](int r, LogitKey k) { top[r] = k.k; });
    for (int r = nc + threadIdx.x; r < a.n; r += kBeamThreads) top[r] = 0;
    if (threadIdx.x == 0) {
      float t = 0.f;
      for (int i = 0; i < kBeamWarps; ++i) t += warp_red[i];
      a.sums[(size_t)row * a.chunks + chunk] = make_float2(m, t);
    }
    __threadfence();
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    is_last = atomicAdd(a.counters + b, 1) == a.beams * a.chunks - 1;
    n_cand = 0;
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();

  // ---- join the request's chunks ----
  // offset[w] = score - log sum of the row; NaN marks a beam that gives no candidates
  for (int i = warp; i < a.beams; i += kBeamWarps) {
    const int r = b * a.beams + i;
    const float score = a.scores[r];
    double off = NAN;
    if (isfinite(score)) {
      const float2* p = a.sums + (size_t)r * a.chunks;
      float m = -INFINITY;
      for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, __ldcg(p + c).x);
      m = warp_max(m);
      if (isfinite(m)) {
        double z = 0.0;
        for (int c = lane; c < a.chunks; c += 32) {
          const float2 q = __ldcg(p + c);
          if (q.x != -INFINITY) z += (double)q.y * exp((double)q.x - (double)m);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        off = (double)score - ((double)m + log(z));
      }
    }
    if (lane == 0) offset[i] = off;
  }
  __syncthreads();
  const int n_lists = a.beams * a.chunks;
  const unsigned long long* tops = a.tops + (size_t)b * n_lists * a.n;
  auto key_of = [&](int list, unsigned long long k) {
    const int i = list / a.chunks;
    const double off = offset[i];
    if (k == 0 || off != off) return BeamKey::none();
    return BeamKey{off + (double)logit_of(k), (uint32_t)(i * a.V + index_of(k))};
  };
  auto entry = [&](int list, int r) -> unsigned long long {  // a dead beam wrote no list
    return offset[list / a.chunks] == offset[list / a.chunks] ? __ldcg(tops + (size_t)list * a.n + r) : 0ull;
  };
  BeamKey mine = BeamKey::none();
  for (int l = threadIdx.x; l < n_lists; l += kBeamThreads) {
    const BeamKey k = key_of(l, entry(l, 0));
    if (k.over(mine)) mine = k;
  }
  const BeamKey edge = block_nth(mine, a.n, sh.j.lists);
  if (!mine.is_none() && !edge.over(mine)) {
    for (int l = threadIdx.x; l < n_lists; l += kBeamThreads)
      for (int r = 0; r < a.n; ++r) {
        const BeamKey k = key_of(l, entry(l, r));
        if (k.is_none() || edge.over(k)) break;
        sh.j.cand[atomicAdd(&n_cand, 1)] = k;
      }
  }
  __syncthreads();
  const int nc = n_cand;
  rank_candidates(sh.j.cand, nc, a.n, [&](int r, BeamKey k) {
    const size_t o = (size_t)b * a.n + r;
    a.out_scores[o] = (float)k.s;
    a.out_beams[o] = (int32_t)(k.at / (uint32_t)a.V);
    a.out_tokens[o] = (int32_t)(k.at % (uint32_t)a.V);
  });
  for (int r = nc + threadIdx.x; r < a.n; r += kBeamThreads) {
    const size_t o = (size_t)b * a.n + r;
    a.out_scores[o] = -INFINITY;
    a.out_beams[o] = -1;
    a.out_tokens[o] = -1;
  }
  if (threadIdx.x == 0) a.counters[b] = 0;
}

bool beam_shape_ok(int B, int beams, int V, int n_out) {
  return B > 0 && B <= kBeamCounterBytes / 4 && beams > 0 && beams <= kMaxBeams && V > 0 && V <= kMaxBeamVocab &&
         n_out > 0 && n_out <= kMaxOut;
}

size_t beam_ws_bytes(int B, int beams, int V, int n_out) {
  const size_t lists = (size_t)B * beams * ((V + kBeamChunk - 1) / kBeamChunk);
  return kBeamCounterBytes + lists * (sizeof(float2) + n_out * sizeof(unsigned long long));
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
  a.beams = beams;
  a.V = V;
  a.n = n_out;
  a.chunks = (V + kBeamChunk - 1) / kBeamChunk;
  a.counters = (int*)workspace;
  a.sums = (float2*)((char*)workspace + kBeamCounterBytes);
  a.tops = (unsigned long long*)(a.sums + (size_t)B * beams * a.chunks);
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  static PerDeviceOnce attr;
  HG_CUDA(attr.run([] {
    return cudaFuncSetAttribute(beam_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(BeamShared));
  }));
  HG_CUDA(launch_pdl(beam_select_kernel, dim3(a.chunks, beams, B), dim3(kBeamThreads), sizeof(BeamShared),
                     (cudaStream_t)stream, a));
  return HIGGS_OK;
}
