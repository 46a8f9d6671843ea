// window_prefill.cu -- paged attention through a sliding window with sinks for prompts, on the
// tcgen05 tensor cores: higgs_window_attention above 64 query rows per kv head (window_attn.cu has
// the mask and the kernel for fewer).
//
// Query rows of one (sequence, kv head) are its tokens x the G query heads of the kv head, flat, so
// G may be any number.  A tile is 256 of them, two halves of 128 (the MMA's M), and walks the keys
// that some row of it sees in blocks of 128: blocks from key 0 for the sinks, then from the page
// where the window of its first token starts.  The kernel is persistent, a CTA per SM taking the
// next tile from a counter, with the rings running on from tile to tile.  The warpgroups:
//   0, 1  softmax, a thread per query row of a half, 64 keys at a time: S_u from tensor memory into
//         registers, mask, maximum and sum, P_u as bf16 over S_u's columns, and O rescaled there
//         when a row's maximum grew by more than 2^8; at the end O / l as bf16 to memory
//   2     loads Q and, alternating, K_j and V_j of 128 keys into 128-byte-swizzled tiles of a ring: by
//         TMA, a box per page, or where a block has keys that no row sees (and whose slots may hold
//         anything: 0 x NaN would be NaN) by 16-byte cp.async with zeros for those
//   3     per half one warp issues S_u = Q K_u^T, two steps ahead, and one O += P_u V_u
// S, P and O of both halves fill the 512 columns of tensor memory: per half two buffers of 64 scores
// and 128 of O.  S_u+1 waits there while the softmax of S_u runs, S_u+2 is issued when P_u V_u is done.
// Both halves share every K and V tile.
//
// P is rounded to bf16: one product per half block and not the two of the decode kernel's hi + lo
// halves, and no columns of tensor memory beyond S's; the weights' errors (2^-9 each, of either sign)
// average out over the keys of a prompt: 0.0023 of the output's norm from the 64-bit result, where the
// rounding of the output alone makes 0.0017 (2048 tokens; 0.0022 and 0.0016 for 8192).
//
// Bound: the serial chain of a softmax warp -- scores from tensor memory, mask, maximum, vote,
// exponentials, pack, store, arrive -- about 1950 cycles per half block of 64 keys and warpgroup; its
// exponentials alone are some 1050 of them (both halves share the SM's 16 a cycle).  B200, 32 / 8
// heads, D = 128, 8192 tokens, window 4096: 0.72 million cycles, that is 369 us at 1965 MHz (1118
// TFLOP/s, 0.65 of a large product's burst rate) and 428 us in a loop of seconds, where the power cap
// holds the clock at 1670 MHz (964 TFLOP/s, 0.67 of the product's sustained rate).  2048 tokens,
// window 1024: 54 us at 1965 MHz, 256 tiles on 148 SMs.  Measured slower for the 8192 tokens, against
// the kernel of the time: 128-row tiles 790 (586); whole 128-key blocks with the product begun early
// 409 (378); the halves half a step apart 380 (378); one warp issuing scores and products 374 (367).
// Few tiles: a tile's keys are not shared out, so a chunk of 17 to 512 tokens (8 to 64 tiles) behind
// 1024 / 4096 / 8192 visible keys takes 26-29 / 70-74 / 129-134 us, all of it one CTA's walk; tiles of
// at most 128 rows run their empty second half too.
// Every mbarrier wait is bounded (about 2 s; the first timeout makes the CTA's other waits give up
// and sets the flag that higgs_tc_error reports; copies and products in flight are then still waited for).
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace higgs {
namespace {

constexpr int kM = 128;          // rows of a half (UMMA M)
constexpr int kTileRows = 2 * kM;
constexpr int kKeys = 128;       // keys of a block, loaded as one tile of K and one of V
constexpr int kHalf = 64;        // keys of half a block: the scores' and weights' unit
constexpr int kWpThreads = 512;  // warpgroups: softmax x 2, loaders, MMA issue
constexpr int kWpTmemCols = 512;
constexpr int kTileRing = 4;     // tile indices handed from the first loader thread to the others
constexpr float kWpSlack = 8.0f;

constexpr uint32_t wp_tile_bytes(int D) { return (uint32_t)kKeys * D * 2; }  // 128 rows of Q, K or V
constexpr int wp_slots(int D) { return D == 128 ? 5 : 8; }
constexpr size_t wp_smem(int D) { return 1024 + (size_t)(2 + wp_slots(D)) * wp_tile_bytes(D); }
static_assert(wp_smem(128) + 1024 <= 227 * 1024, "shared memory budget");

struct WpArgs {
  const uint16_t* q;
  const uint16_t* kc;
  const uint16_t* vc;
  int64_t page_stride, head_stride;
  const int32_t* bt;
  int max_blocks;
  const int32_t* seq_lens;
  int B, Lq, Hq, Hkv, G, window, sinks;
  int q_tiles, tiles;  // tiles of a (sequence, kv head); of the launch
  float scale_log2;
  uint16_t* out;
  int* err;
  int* counters;  // [0] tiles taken, [1] CTAs done: zero before the launch and after it
};

// Tile i: rows [r0, r_end) of (sequence, kv head) i % (B Hkv), later rows first; its blocks are
// `sink_blocks` from key 0 for keys < sink_keys, then those from `base` up to kv_len.
struct WpTile {
  int b, h, r0, r_end, first, kv_len, lo, base, sink_keys, sink_blocks, blocks;
  __device__ WpTile(const WpArgs& a, int i) {
    const int bh = a.B * a.Hkv, qt = i / bh, p = i - qt * bh;
    b = p / a.Hkv;
    h = p - b * a.Hkv;
    r0 = (a.q_tiles - 1 - qt) * kTileRows;
    r_end = min(a.Lq * a.G, r0 + kTileRows);
    first = a.seq_lens[b] - a.Lq;  // position of query token 0
    kv_len = max(0, min(first + (r_end - 1) / a.G + 1, a.max_blocks * 16));
    lo = max(0, max(0, first + r0 / a.G) - a.window + 1);
    base = lo & ~15;
    sink_keys = min(a.sinks, base);
    sink_blocks = kv_len > 0 ? (sink_keys + kKeys - 1) / kKeys : 0;
    blocks = kv_len > 0 ? sink_blocks + (kv_len - base + kKeys - 1) / kKeys : 0;
  }
  __device__ bool is_sink(int j) const { return j < sink_blocks; }
  __device__ int key(int j) const { return is_sink(j) ? j * kKeys : base + (j - sink_blocks) * kKeys; }
  __device__ int keys_end(int j) const { return is_sink(j) ? sink_keys : kv_len; }
  // half blocks of 64 keys that hold any key: 2, or 1 of the last block of either part
  __device__ int halves(int j) const { return keys_end(j) - key(j) > kHalf ? 2 : 1; }
};

__device__ __forceinline__ bool wp_wait(uint64_t* bar, unsigned parity, volatile int* abort, int* err) {
  const uint32_t a = smem_u32(bar);
  const long long t0 = clock64();
  for (unsigned it = 0;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 63) == 63) {
      if (*abort) return false;
      if (clock64() - t0 > (1ll << 32)) break;  // ~2 s at 2 GHz
    }
  }
  *abort = 1;
  atomicExch(err, 1);
  return false;
}

__device__ __forceinline__ float wp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint32_t pack_p(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One lane of the warp, the same each time.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred;
}

// tcgen05 instructions of the elected lane in code that the whole warp runs: operands that are the
// same for all lanes then sit in uniform registers, which these instructions take, and each costs
// an issue slot; under a branch of one lane they are moved there first, operand by operand.
// A descriptor's shared-memory address moved on by `bytes`: the field holds addresses of up to 256
// KB without a carry.
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) {
  return (desc & 0xffffffff00000000ull) | ((uint32_t)desc + (bytes >> 4));
}

__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accum), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accum), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}

__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int d, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(d), "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

template <int D>
__global__ void __launch_bounds__(kWpThreads, 1)
    window_prefill_kernel(WpArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  constexpr int SLOTS = wp_slots(D), DC = D / 8;  // DC: 16-byte chunks of a row
  constexpr uint32_t kTile = wp_tile_bytes(D);
  constexpr int COL_O = 2 * kM;  // S (and P over it) of half x, buffer u & 1, at 128 x + 64 (u & 1); O at 256 + 128 x
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = smem;               // [half][D / 64 panels][128 rows][128 B], 128-byte swizzle
  uint8_t* ring = smem + 2 * kTile;  // K_0, V_0, K_1, ... of all the CTA's tiles: [D / 64][128 keys][128 B]
  __shared__ __align__(8) uint64_t q_full, q_empty;                     // a phase per tile
  __shared__ __align__(8) uint64_t kv_full[SLOTS], kv_empty[SLOTS];
  __shared__ __align__(8) uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [half][buffer]
  __shared__ __align__(8) uint64_t o_free[2];                           // a phase per tile
  __shared__ __align__(8) uint64_t t_full[kTileRing], t_empty[kTileRing];
  __shared__ int tile_ring[kTileRing];
  __shared__ __align__(8) uint64_t drained;
  __shared__ int loader_tile, abort_flag, drain_abort;
  __shared__ uint32_t tmem_base;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = warp >> 2;
  volatile int* abort = &abort_flag;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 4);
    mbar_init(&q_empty, 2);
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&kv_full[s], 4);
      mbar_init(&kv_empty[s], 2);
    }
    for (int x = 0; x < 2; ++x) {
      for (int u = 0; u < 2; ++u) {
        mbar_init(&s_full[x][u], 1);
        mbar_init(&p_full[x][u], 128);
        mbar_init(&pv_done[x][u], 1);
      }
      mbar_init(&o_free[x], 128);
    }
    for (int i = 0; i < kTileRing; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], 256 + 4);
    }
    mbar_init(&drained, 4);
    abort_flag = drain_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  if (warp == 12) {
    tc_alloc(&tmem_base, kWpTmemCols);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = tmem_base;
  pdl_launch();

  // the tile of round k for the softmax threads and the issuing warps (`tiles` once none is left)
  auto next_tile = [&](int k, bool arrive) {
    wp_wait(&t_full[k % kTileRing], (k / kTileRing) & 1, abort, a.err);
    const int i = *abort ? a.tiles : *(volatile int*)&tile_ring[k % kTileRing];
    const int same = __shfl_sync(0xffffffffu, i, 0);  // one answer for the warp, read by all before ...
    if (arrive) mbar_arrive(&t_empty[k % kTileRing]);  // ... the slot is free
    return same;
  };

  if (group == 2) {
    // ---------------- loaders ----------------
    const int lt = threadIdx.x - 256;
    constexpr int KSTEP = 128 / DC, KPT = kKeys / KSTEP;  // rows of a tile per thread, KSTEP apart
    const int dc = lt % DC, k0 = lt / DC;
    static_assert(KSTEP % 8 == 0, "a thread's rows share their swizzle");
    const uint32_t so = (dc >> 3) * (kKeys * 128) + k0 * 128 + (((dc & 7) ^ (k0 & 7)) << 4);
    const uint32_t q_addr = smem_u32(qs) + so, ring_addr = smem_u32(ring) + so;
    int n = 0, k = 0;  // ring tiles issued; tiles taken
    for (;; ++k) {
      if (lt == 0) {
        int i = k == 0 ? blockIdx.x : gridDim.x + atomicAdd(a.counters, 1);
        if (i > a.tiles || *abort) i = a.tiles;
        if (k >= kTileRing) wp_wait(&t_empty[k % kTileRing], ((k / kTileRing) - 1) & 1, abort, a.err);
        *(volatile int*)&tile_ring[k % kTileRing] = i;
        mbar_arrive(&t_full[k % kTileRing]);
        loader_tile = i;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const int i = loader_tile;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (i >= a.tiles) break;
      const WpTile T(a, i);
      const int32_t* bt = a.bt + (size_t)T.b * a.max_blocks;
      const size_t col = (size_t)T.h * a.head_stride + dc * 8;
      for (int j = 0; j < max(1, T.blocks); ++j) {
        const int kb = T.key(j);
        // a block all of whose keys are seen by some row comes by TMA, a box per page and 64 of d
        const bool whole = kb + kKeys <= T.keys_end(j) && (T.is_sink(j) || kb >= T.lo || kb + kKeys <= a.sinks);
        const int n0 = n;
        if (j < T.blocks && whole) {
          const int box = lane % (8 * (D / 64)), page = bt[(kb >> 4) + box / (D / 64)], panel = box % (D / 64);
#pragma unroll
          for (int v = 0; v < 2; ++v, ++n) {
            const int s = n % SLOTS;
            if (n >= SLOTS) wp_wait(&kv_empty[s], ((n / SLOTS) - 1) & 1, abort, a.err);
            __syncwarp();
            if (lane == 0) {
              if (warp == 8)
                mbar_arrive_expect_tx(&kv_full[s], kTile);
              else
                mbar_arrive(&kv_full[s]);
            }
            __syncwarp();
            if (warp == 8 && lane < 8 * (D / 64))
              tma_page(smem_u32(ring) + s * kTile + panel * (kKeys * 128) + (box / (D / 64)) * 2048,
                       v ? &v_map : &k_map, panel * 64, T.h, page, &kv_full[s]);
          }
        } else if (j < T.blocks) {
          int64_t off[KPT];  // < 0: a key that no row sees; its page is not looked up, it may be free
#pragma unroll
          for (int q = 0; q < KPT; ++q) {
            const int kg = kb + k0 + q * KSTEP;
            const bool ok = kg < T.keys_end(j) && (T.is_sink(j) || kg >= T.lo || kg < a.sinks);
            off[q] = ok ? (int64_t)bt[kg >> 4] * a.page_stride + (int64_t)col + (kg & 15) * D : -1;
          }
#pragma unroll
          for (int v = 0; v < 2; ++v, ++n) {
            const int s = n % SLOTS;
            if (n >= SLOTS) wp_wait(&kv_empty[s], ((n / SLOTS) - 1) & 1, abort, a.err);
            const uint16_t* pool = v ? a.vc : a.kc;
#pragma unroll
            for (int q = 0; q < KPT; ++q)
              cp_async16_or_zero(ring_addr + s * kTile + q * KSTEP * 128, pool + (off[q] < 0 ? 0 : off[q]), off[q] >= 0);
          }
        }
        if (j == 0) {
          // Q, once the tile before has had its last scores (the first K and V are on their way)
          if (k >= 1) wp_wait(&q_empty, (k - 1) & 1, abort, a.err);
#pragma unroll 4
          for (int r = k0; r < kTileRows; r += KSTEP) {
            const int rr = T.r0 + r, t = rr / a.G, hd = rr - t * a.G;
            const bool ok = rr < T.r_end;
            const uint16_t* src = a.q + (((size_t)T.b * a.Lq + (ok ? t : 0)) * a.Hq + T.h * a.G + hd) * D + dc * 8;
            cp_async16_or_zero(q_addr + (r >> 7) * kTile + ((r & 127) - k0) * 128, src, ok);
          }
        }
        if (j == 0 || (j < T.blocks && !whole)) {
          // the copies are in shared memory: generic writes before the tensor core's reads
          cp_async_commit();
          cp_async_wait<0>();
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if (j < T.blocks && !whole) {
              mbar_arrive(&kv_full[n0 % SLOTS]);
              mbar_arrive(&kv_full[(n0 + 1) % SLOTS]);
            }
            if (j == 0) mbar_arrive(&q_full);
          }
        }
      }
    }
    // No copy and no arrival may come after the CTA's shared memory is another's: the ring's copies
    // (also those that nobody waited for because a wait gave up), then the products' releases.
    for (int e = max(0, n - SLOTS); e < n; ++e)
      wp_wait(&kv_full[e % SLOTS], (e / SLOTS) & 1, &drain_abort, a.err);
    for (int e = max(0, n - SLOTS); e < n; ++e) wp_wait(&kv_empty[e % SLOTS], (e / SLOTS) & 1, abort, a.err);
    if (k >= 1) wp_wait(&q_empty, (k - 1) & 1, abort, a.err);
  } else if (group == 3) {
    // ---------------- MMA issue: scores of half x by warp 12 + x, products by warp 14 + x ----------------
    // (One warp for both holds the next product back behind the next scores.)
    const int x = warp & 1;
    const uint32_t lead = elect_lane();
    const uint32_t ub = __shfl_sync(0xffffffffu, tb, 0);
    const uint32_t col_s = ub + x * kM, col_o = ub + COL_O + x * kM;
    // blocks and half blocks of the CTA's tiles so far: K and V of block J are ring tiles 2 J and
    // 2 J + 1, half block U has buffer U & 1 of tensor memory
    int J = 0, U = 0;
    for (int k = 0;; ++k) {
      const int i = next_tile(k, lead != 0);
      if (i >= a.tiles) break;
      const WpTile T(a, i);
      if (warp < 14) {
        constexpr uint32_t id = tc_idesc_bf16(kM, kHalf);
        const uint64_t q_desc = sw128_desc(smem_u32(qs) + x * kTile), k_desc = sw128_desc(smem_u32(ring));
        wp_wait(&q_full, k & 1, abort, a.err);
        for (int j = 0; j < T.blocks; ++j, ++J) {
          const int slot = (2 * J) % SLOTS, nh = T.halves(j);
          wp_wait(&kv_full[slot], ((2 * J) / SLOTS) & 1, abort, a.err);
          for (int h = 0; h < nh; ++h, ++U) {
            // S_u = Q K_u^T into the buffer that holds P_{u-2} until its product is done
            if (U >= 2) wp_wait(&pv_done[x][U & 1], ((U >> 1) - 1) & 1, abort, a.err);
            tc_fence_after();
            const uint64_t kd = desc_at(k_desc, slot * kTile + h * (kHalf * 128));
            const uint32_t cs = col_s + (U & 1) * kHalf;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_ss(lead, cs, desc_at(q_desc, (kk >> 2) * (kM * 128) + (kk & 3) * 32),
                     desc_at(kd, (kk >> 2) * (kKeys * 128) + (kk & 3) * 32), id, kk > 0);
            commit_if(lead, &s_full[x][U & 1]);
          }
          commit_if(lead, &kv_empty[slot]);
        }
        commit_if(lead, &q_empty);  // (at once if the tile had no block)
      } else {
        constexpr uint32_t id = tc_idesc_bf16(kM, D, true);
        const uint64_t v_desc = sw128_mn_desc(smem_u32(ring), kKeys * 128);
        for (int j = 0; j < T.blocks; ++j, ++J) {
          const int slot = (2 * J + 1) % SLOTS, nh = T.halves(j);
          wp_wait(&kv_full[slot], ((2 * J + 1) / SLOTS) & 1, abort, a.err);
          // a tile's first product overwrites O: its threads have read the tile's before
          if (j == 0 && k >= 1) wp_wait(&o_free[x], (k - 1) & 1, abort, a.err);
          for (int h = 0; h < nh; ++h, ++U) {
            wp_wait(&p_full[x][U & 1], (U >> 1) & 1, abort, a.err);
            tc_fence_after();
            const uint64_t vd = desc_at(v_desc, slot * kTile + h * (kHalf * 128));
            const uint32_t cs = col_s + (U & 1) * kHalf;
#pragma unroll
            for (int kk = 0; kk < kHalf / 16; ++kk)  // 16 keys = two 8-row atoms = 2 KB
              mma_ts(lead, col_o, cs + kk * 8, desc_at(vd, kk * 2048), id, j > 0 || h > 0 || kk > 0);
            commit_if(lead, &pv_done[x][U & 1]);
          }
          commit_if(lead, &kv_empty[slot]);
        }
      }
    }
    // tensor memory is given back after the last product, also when a wait gave up before it
    commit_if(lead, &drained);
    wp_wait(&drained, 0, &drain_abort, a.err);
  } else {
    // ---------------- softmax: half x, a thread per row ----------------
    const int x = group, r = x * kM + (threadIdx.x & 127);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t col_s = tb + lanes + x * kM, col_o = tb + lanes + COL_O + x * kM;
    const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
    int U = 0;
    for (int k = 0;; ++k) {
      const int i = next_tile(k, true);
      if (i >= a.tiles) break;
      const WpTile T(a, i);
      const int rr = T.r0 + r, t = rr / a.G, hd = rr - t * a.G;
      const bool valid = rr < T.r_end;
      const int pos = valid ? T.first + t : -1;
      float m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      const int u0 = U;
      for (int j = 0, h = 0; j < T.blocks; ++U) {
        const int buf = U & 1, phase = (U >> 1) & 1;
        const uint32_t cs = col_s + buf * kHalf;
        wp_wait(&s_full[x][buf], phase, abort, a.err);
        tc_fence_after();
        float v[kHalf];
#pragma unroll
        for (int c = 0; c < kHalf / 16; ++c) tc_ld16(cs + 16 * c, v + 16 * c);
        // key i of the half block is visible iff i <= lim and (i >= low or i < snk)
        const int kb = T.key(j) + h * kHalf;
        const int lim = (T.is_sink(j) ? min(pos, T.sink_keys - 1) : pos) - kb;
        if (++h == T.halves(j)) {
          h = 0;
          ++j;
        }
        const int low = pos - a.window + 1 - kb, snk = a.sinks - kb;
        const bool whole = __all_sync(0xffffffffu, lim >= kHalf - 1 && (low <= 0 || snk >= kHalf));
        tc_wait_ld();
        if (!whole) {
          auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
#pragma unroll
          for (int c = 0; c < kHalf / 32; ++c) {
            const uint32_t vis = below(lim + 1 - 32 * c) & (~below(low - 32 * c) | below(snk - 32 * c));
#pragma unroll
            for (int q = 0; q < 32; ++q) v[32 * c + q] = (vis >> q) & 1u ? v[32 * c + q] : -INFINITY;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < kHalf; q += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx4[e] = fmaxf(mx4[e], fmaxf(v[q + e], v[q + 4 + e]));
        // raw scores: the scale (> 0) is applied to the maximum and folded into the exponent's FMA
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
        const bool grow = mx > m + kWpSlack || (m == -INFINITY && mx != -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? wp_ex2(m - mx) : 1.f;  // m = -inf: 0 (O and l hold zeros)
          if (grow) m = mx;
          l2.x *= alpha;
          l2.y *= alpha;
          if (U > u0) {
            wp_wait(&pv_done[x][buf ^ 1], ((U - 1) >> 1) & 1, abort, a.err);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              float o[16];
              tc_ld16(col_o + 16 * c, o);
              tc_wait_ld();
              uint32_t w[16];
#pragma unroll
              for (int q = 0; q < 16; ++q) w[q] = __float_as_uint(o[q] * alpha);
              tc_st16(col_o + 16 * c, w);
            }
          }
        }
        const float mm = m == -INFINITY ? 0.f : m;  // (nothing visible yet: every score is -inf)
        const float2 neg_m = make_float2(-mm, -mm);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < kHalf / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 e = __ffma2_rn(make_float2(v[32 * c + 2 * q], v[32 * c + 2 * q + 1]), scale2, neg_m);
            const float2 p = make_float2(wp_ex2(e.x), wp_ex2(e.y));
            sum[q & 1] = __fadd2_rn(sum[q & 1], p);
            pk[q] = pack_p(p.x, p.y);
          }
          tc_st16(cs + 16 * c, pk);
        }
        l2 = __fadd2_rn(l2, __fadd2_rn(sum[0], sum[1]));
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[x][buf]);
      }
      // ---- O / l -> bf16 ----
      if (T.blocks > 0) {
        wp_wait(&pv_done[x][(U - 1) & 1], ((U - 1) >> 1) & 1, abort, a.err);
        tc_fence_after();
      }
      const float l = l2.x + l2.y, inv = l > 0.f ? 1.f / l : 0.f;
      uint16_t* dst = a.out + (((size_t)T.b * a.Lq + t) * a.Hq + T.h * a.G + hd) * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (T.blocks > 0) {
          tc_ld16(col_o + 32 * c, o);
          tc_ld16(col_o + 32 * c + 16, o + 16);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int q = 0; q < 32; ++q) o[q] = 0.f;
        }
        if (valid) {
#pragma unroll
          for (int q = 0; q < 32; q += 8)
            *reinterpret_cast<uint4*>(dst + 32 * c + q) =
                make_uint4(pack_p(o[q] * inv, o[q + 1] * inv), pack_p(o[q + 2] * inv, o[q + 3] * inv),
                           pack_p(o[q + 4] * inv, o[q + 5] * inv), pack_p(o[q + 6] * inv, o[q + 7] * inv));
        }
      }
      tc_fence_before();
      mbar_arrive(&o_free[x]);  // the next tile's first product may overwrite O
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tc_dealloc(tb, kWpTmemCols);
  }
  if (threadIdx.x == 0) {  // the last CTA to finish leaves the counters at zero
    __threadfence();
    if (atomicAdd(a.counters + 1, 1) == (int)gridDim.x - 1) {
      a.counters[0] = 0;
      a.counters[1] = 0;
      __threadfence();
    }
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A pool as [pages, kv heads, 16, D], in boxes of one head's page by 64 of d, 128-byte swizzle.
bool pool_map(const void* pool, int Hkv, int D, int64_t page_stride, int64_t head_stride, CUtensorMap* out) {
  static EncodeFn encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeFn>(p)
               : nullptr;
  }();
  if (!encode) return false;
  // (the number of pages is not known here: ids come from the block table; the stride of a
  // dimension of one head is never used)
  const cuuint64_t dims[4] = {(cuuint64_t)D, HIGGS_PAGE_SIZE, (cuuint64_t)Hkv, (cuuint64_t)INT32_MAX};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2,
                                 Hkv == 1 ? (cuuint64_t)D * 2 * HIGGS_PAGE_SIZE : (cuuint64_t)head_stride * 2,
                                 (cuuint64_t)page_stride * 2};
  const cuuint32_t box[4] = {64, HIGGS_PAGE_SIZE, 1, 1}, step[4] = {1, 1, 1, 1};
  return encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch_wp(const WpArgs& a, cudaStream_t st) {
  CUtensorMap k_map, v_map;
  if (!pool_map(a.kc, a.Hkv, D, a.page_stride, a.head_stride, &k_map) ||
      !pool_map(a.vc, a.Hkv, D, a.page_stride, a.head_stride, &v_map))
    return cudaErrorInvalidValue;
  auto k = window_prefill_kernel<D>;
  static PerDeviceOnce attr;
  const cudaError_t e =
      attr.run([&] { return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wp_smem(D)); });
  if (e != cudaSuccess) return e;
  return launch_pdl(k, dim3(std::min(a.tiles, sm_count())), dim3(kWpThreads), wp_smem(D), st, a, k_map, v_map);
}

}  // namespace

cudaError_t launch_window_prefill(const void* q, int B, int Lq, int Hq, int Hkv, int D, const void* kc, const void* vc,
                                  int64_t page_stride, int64_t head_stride, const int32_t* bt, int max_blocks,
                                  const int32_t* seq_lens, int window, int sinks, float scale, void* out,
                                  int* counters, int* err, cudaStream_t st) {
  WpArgs a;
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)kc;
  a.vc = (const uint16_t*)vc;
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  a.bt = bt;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.B = B;
  a.Lq = Lq;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.window = window;
  a.sinks = sinks;
  a.q_tiles = (Lq * a.G + kTileRows - 1) / kTileRows;
  a.tiles = a.q_tiles * B * Hkv;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (uint16_t*)out;
  a.err = err;
  a.counters = counters;
  return D == 64 ? launch_wp<64>(a, st) : launch_wp<128>(a, st);
}

}  // namespace higgs
