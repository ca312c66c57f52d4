// Attention of packed prompts on the tcgen05 tensor cores.  Rules: include/uniql_b200.h.
//
// Mathematics: one pass over the keys with a running bound m of the row's scores (in units of log2): with S = Q K^T and f =
// softmax_scale log2(e), P = 2^(f S - m), l = sum P, O = sum P V, and O / l at the end.  m is raised, and l and O rescaled, only
// when a score exceeds it by more than 8 (P stays below 2^8, far from fp16's limit), which after the first tiles is rare.
//
// A CTA owns two units, a unit being 128 query rows: 128 tokens of one query head, or 128 / group tokens of all query heads of a
// kv head.  Units of a request and kv head are numbered row block first, head of the group second, so that the two share their keys
// and values.  Per 128 keys and unit:
//   S (tensor memory, 128 fp32 columns) = Q (shared memory) K^T (shared memory)
//   P (16-bit, on the first 64 of S's columns) -- four softmax warps, one row a thread
//   O (tensor memory) += P V, P read from tensor memory, V as an MN-major operand straight from its row-major tile
// While the softmax of one unit runs the tensor cores work on the other:  warps 0-3 and 4-7 softmax of unit 0 and 1 (they also
// rescale and store O), warp 8 issues the MMAs, warp 9 the TMA loads (no multicast), warp 10 hands out the items.
// Few units (at most one an SM) are items of their own: 256 tokens of 28 heads 8.8 us, 12.6 as pairs on half of the SMs.
//
// P has the input type because one product takes two operands of one type; its sum l is taken in fp32 before that.  Each term is off by
// half a step of the type: error against 64 bits 1.2 to 1.4 times that of fp32 arithmetic, whose results are rounded alike.
//
// (Pairs of times below are short bursts of the kernel as it was when that step was made; they compare with each other alone.)
// A thread stores 32 bytes of its row at a time: every store instruction touches 32 rows, which takes the load/store unit 32
// cycles whatever their width (16 packed prompts: 497 us with 16 bytes at a time, 480 with 32).
//
// Items.  A CTA stays on its SM and takes one pair of units after the other, by cluster launch control (the grid names every item;
// a running CTA asks for the place of one that has not begun).  The next item's queries, keys and first scores then run under
// the end of the one before, and the items even out over the SMs: 16 packed prompts 515 us against 562 as one CTA an item, and
// 548 when every CTA takes every 148th (9.6 % uneven there; all three with stores of 16 bytes).
//
// Masked places: keys behind a request's last are set to -inf in S, and the rows of V behind it in its last tile, which belong
// to another request, are cleared in shared memory before they are multiplied by the zeros of P.
// Bound: 128 keys of both units cost 2048 cycles of MMA, 2048 of shared memory traffic (Q and K are both read from there) and 2048
// of exponentials (16 a clock and SM); they take 3135, the rest being the hops S -> softmax -> P -> O of a unit that the other
// unit's work does not cover, at the 1.6 GHz that the part's power limit leaves (16384 tokens, 32 heads of 128, fp16, causal: 1.8 ms
// in a short burst, 1.98 ms back to back = 1.11 PFLOP/s; 16 packed prompts of up to 2048 tokens, all behind a prefix: 541 us back to
// back = 0.94 PFLOP/s of visible pairs).  Tried without gain: S in two 64-key buffers a unit (Q is read twice as
// often: 2.07 ms against 1.79), P handed over in quarters (1.83 to 2.0), a quarter of the exponentials as polynomials on the FMA
// pipe (1.75 to 1.96), waits polled without a suspend time (2.00 against 2.05 back to back).  These were measured with one CTA an item.
// Every wait is bounded; a wait that gives up sets UNIQL_STATUS_WAIT_TIMEOUT and the kernel drains.
#include "common.cuh"
#include "kv_cache.cuh"
#include "tc.cuh"

namespace uniql {

namespace pa {
constexpr int kMmaWarp = 8, kLoadWarp = 9, kPlanWarp = 10;        // warps 0-7: softmax
constexpr int kThreads = 384;                   // three warpgroups; the third has an idle warp
constexpr int kSoftmaxRegs = 208, kOtherRegs = 80;      // 2 * 208 + 80 <= 3 * 168, what the block is launched with
constexpr int kRows = 128, kKeys = 128;
constexpr int kTmemCols = 512;                  // S0, S1, O0, O1: 128 columns each
// Barriers that say "rows of other requests cleared", taken in turn.  One would not do: the load warp may clear the next item's last
// tile before the MMA thread has seen this one's phase, whose parity would then never come.  With two, clearing c + 2 waits for the
// queries of the item behind that of clearing c (bar_qfree), which the MMA thread frees only behind its wait for clearing c.
constexpr int kCleans = 2;
template <int DP>
struct Cfg {
  static constexpr int kTileBytes = 128 * DP * 2;
  static constexpr int kStages = 5;
  static constexpr int kOffKv = 2 * kTileBytes;
  static constexpr int kOffBar = kOffKv + kStages * kTileBytes;
  static constexpr int kBars = 1 + 2 * kStages + 2 + 4 + 2 + kCleans + 1 + 2 + 2 + 2 + 1 + 1;
  static constexpr int kSmem = kOffBar + kBars * 8 + 16 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};
}  // namespace pa

// Cluster launch control: ask for the place of a CTA of this grid that has not begun, and read the answer (16 bytes, behind `bar`).
__device__ __forceinline__ void pa_ask_next(uint32_t answer, uint32_t bar) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool pa_next(uint32_t answer, long long& x) {
  uint32_t ok, at = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(ok), "=r"(at)
      : "r"(answer)
      : "memory");
  x = at;
  return ok != 0;
}

// What a CTA works on at a time: two units of a request and kv head.
struct PaItem {
  int kvh;                                      // -1: no more
  int q0, nq, k0, nk;                           // the request's rows
  int row[2], head[2], n[2];                    // of each unit: first query row, query head (-1: none), tiles of keys
};

struct PaParams {
  const int32_t* cu_q;
  const int32_t* cu_k;
  unsigned char* out;
  int* status_word;
  int batch, total_q, total_k, heads, kv_heads, group, dk, dv, causal;
  int units;                                    // of an item: 2, or 1
  int pack, tokens;                             // of a unit: query heads (1, or the whole group) and tokens (128 / pack)
  int parts;                                    // group / pack: units of a row block and kv head
  int wide;                                     // rows of the result are 32-byte aligned
  float scale_log2;
};

__device__ __forceinline__ void pa_tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pa_ld32(uint32_t taddr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
        "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
        "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]),
        "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
__device__ __forceinline__ void pa_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_st32(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]),
        "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]),
        "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]),
        "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
__device__ __forceinline__ void pa_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pa_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pa_st16(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]),
        "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void pa_store32(void* at, const uint32_t* x) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]),
               "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
               : "memory");
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {   // NaN if any is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pa_pack(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(pa::kThreads, 1)
prompt_attention_kernel(const __grid_constant__ PaParams p, const __grid_constant__ CUtensorMap qmap,
                        const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using namespace pa;
  using C = Cfg<DP>;
  constexpr int SUB = 128 * 128;                // bytes of a sub-tile of 128 rows x 64 channels
  extern __shared__ uint8_t smem_unaligned[];
  __shared__ PaItem s_item[2];
  __shared__ __align__(16) uint4 s_next[2];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = tc_smem_addr(smem);
  const uint32_t bar_q = sbase + C::kOffBar, bar_full = bar_q + 8, bar_empty = bar_full + 8 * C::kStages;
  const uint32_t bar_s = bar_empty + 8 * C::kStages, bar_p = bar_s + 16, bar_o = bar_p + 32, bar_clean = bar_o + 16;
  const uint32_t bar_qfree = bar_clean + 8 * kCleans, bar_ofree = bar_qfree + 8, bar_item = bar_ofree + 16, bar_taken = bar_item + 16, bar_next = bar_taken + 16, bar_loaded = bar_next + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::kOffBar + C::kBars * 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_addr((const void*)tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kLoadWarp && tc_elect()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    tc_mbar_init(bar_q, 1);
    for (int s = 0; s < C::kStages; ++s) {
      tc_mbar_init(bar_full + 8 * s, 1);
      tc_mbar_init(bar_empty + 8 * s, 1);
    }
    for (int t = 0; t < 2; ++t) {
      tc_mbar_init(bar_s + 8 * t, 1);
      tc_mbar_init(bar_p + 16 * t, 4);          // the first 64 columns of P, then the others
      tc_mbar_init(bar_p + 16 * t + 8, 4);
      tc_mbar_init(bar_o + 8 * t, 1);
    }
    for (int t = 0; t < kCleans; ++t) tc_mbar_init(bar_clean + 8 * t, 1);
    tc_mbar_init(bar_qfree, 1);
    tc_mbar_init(bar_next, 1);
    tc_mbar_init(bar_loaded, 1);
    for (int t = 0; t < 2; ++t) {
      tc_mbar_init(bar_ofree + 8 * t, 4);
      tc_mbar_init(bar_item + 8 * t, 1);
      tc_mbar_init(bar_taken + 8 * t, 2 + kMmaWarp);           // load warp, MMA thread, softmax warps
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  auto begin_q = [&](int b) { return min(max(p.cu_q[b], 0), p.total_q); };
  auto begin_k = [&](int b) { return min(max(p.cu_k[b], 0), p.total_k); };
  // a request whose rows all exist; one that is not has no keys: with some of its rows cut off its queries would see the wrong ones
  auto sound = [&](int b) {
    const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
    return 0 <= q0 && q0 <= q1 && q1 <= p.total_q && 0 <= k0 && k0 <= k1 && k1 <= p.total_k;
  };
  // behind the last key of all the loads fill in zeros by themselves
  auto dirty = [&](const PaItem& w, int tiles) { return tiles * kKeys > w.nk && w.k0 + w.nk < p.total_k; };
  const uint32_t tmem = *tmem_slot;
  bool timed_out = false;
  // The items of a CTA, one behind the other: every role walks them by itself.  item(k): the k-th one, false behind the last or when a
  // wait of the role has given up; a warp decides that together.
  auto item = [&](int k, PaItem& w, bool whole_warp) {
    if (!timed_out && !tc_mbar_wait(bar_item + 8 * (k & 1), (k >> 1) & 1)) timed_out = true;
    if (whole_warp) timed_out = __any_sync(~0u, timed_out);
    if (timed_out) return false;
    w = s_item[k & 1];
    return w.kvh >= 0;
  };

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kPlanWarp) {
      // ------------------------------------------------------------------ items: pairs of units of all requests in order, kv head
      // fastest, the last row blocks (the ones with the most keys) of a request first.  The grid has a CTA for every item; one
      // that runs takes the places of others that have not begun (cluster launch control), so that the next item's loads and
      // products start while the last one's results are written, and whoever is free first takes the next item.
      auto pairs_of = [&](int b) {
        const int n = max(begin_q(b + 1) - begin_q(b), 0);
        return (long long)(((n + p.tokens - 1) / p.tokens) * (long long)p.parts + p.units - 1) / p.units;
      };
      const int per = (p.batch + 31) / 32;
      const int b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
      long long mine = 0;
      bool bad = false;                         // requests whose queries do not all exist, and below, of those with rows, keys
      for (int b = b0; b < b1; ++b) {
        mine += pairs_of(b);
        bad |= p.cu_q[b] < 0 || p.cu_q[b + 1] < p.cu_q[b] || p.cu_q[b + 1] > p.total_q;
      }
      long long incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += v;
      }
      const long long before = incl - mine, total = __shfl_sync(~0u, incl, 31) * p.kv_heads;
      const int low = p.batch > 0 ? begin_q(0) : p.total_q, high = p.batch > 0 ? begin_q(p.batch) : p.total_q;
      long long x = blockIdx.x;
      bool more = true;
      for (int k = 0;; ++k) {
        if (more)                               // rows that no request owns: cleared by the way
          for (long long r = x; r < low + p.total_q - high; r += gridDim.x) {
            uint4* dst = reinterpret_cast<uint4*>(p.out + (size_t)(r < low ? r : r - low + high) * p.heads * p.dv * 2);
            for (int i = lane; i < p.heads * p.dv / 8; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
          }
        if (k >= 2 && !timed_out && !tc_mbar_wait(bar_taken + 8 * (k & 1), ((k >> 1) & 1) ^ 1)) timed_out = true;
        timed_out = __any_sync(~0u, timed_out);
        if (timed_out) break;                   // the others give up by themselves
        const long long pair = x / p.kv_heads;
        PaItem w;
        if (more && x < total) {
          // the lane whose requests hold the pair works the item out
          const bool hit = before <= pair && pair < before + mine;
          if (hit) {
            long long at = before, n = 0;
            int b = b0;
            for (; b < b1; ++b) {
              n = pairs_of(b);
              if (pair < at + n) break;
              at += n;
            }
            w.kvh = (int)(x - pair * p.kv_heads);
            w.q0 = begin_q(b);
            w.nq = begin_q(b + 1) - w.q0;
            w.k0 = begin_k(b);
            const bool all = sound(b);
            bad |= !all;
            w.nk = all ? begin_k(b + 1) - w.k0 : 0;
            const int units = ((w.nq + p.tokens - 1) / p.tokens) * p.parts, u0 = p.units * (int)(n - 1 - (pair - at));
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int u = t < p.units ? u0 + t : units;
              const int row = u / p.parts * p.tokens;
              int seen = w.nk;                  // query i sees the keys below i + 1 + nk - nq
              if (p.causal) seen = min(w.nk, max(min(row + p.tokens, w.nq) + w.nk - w.nq, 0));
              w.row[t] = row;
              w.head[t] = u < units ? w.kvh * p.group + u % p.parts * p.pack : -1;
              w.n[t] = u < units ? (seen + kKeys - 1) / kKeys : 0;
            }
            s_item[k & 1] = w;
          }
        } else if (lane == 0) {                 // none behind this one, or a place of the grid that is no item
          s_item[k & 1].kvh = more ? 0 : -1;
          s_item[k & 1].n[0] = s_item[k & 1].n[1] = 0;
          s_item[k & 1].head[0] = s_item[k & 1].head[1] = -1;
        }
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(bar_item + 8 * (k & 1));
        if (!more) break;
        // the next one is asked for when this one's loads have all been issued: earlier, it could be another CTA's sooner
        if (!tc_mbar_wait(bar_loaded, k & 1)) timed_out = true;
        timed_out = __any_sync(~0u, timed_out);
        if (timed_out) break;
        if (lane == 0) pa_ask_next(tc_smem_addr(&s_next[k & 1]), bar_next);
        if (!tc_mbar_wait(bar_next, k & 1)) timed_out = true;
        timed_out = __any_sync(~0u, timed_out);
        if (timed_out) break;
        more = pa_next(tc_smem_addr(&s_next[k & 1]), x);
      }
      if (bad && p.status_word) atomicOr(p.status_word, UNIQL_STATUS_BAD_INDEX);
    }
    if (warp == kLoadWarp) {
      // ------------------------------------------------------------------ loads: Q, then K 0, V 0, K 1, V 1, ... of every item
      PaItem w;
      int it0 = 0, qs = 0, cleans = 0;          // tiles and items loaded, tiles cleared so far
      for (int k = 0; item(k, w, true); ++k) {
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(bar_taken + 8 * (k & 1));
        const int nmax = max(w.n[0], w.n[1]);
        if (nmax == 0) {
          if (lane == 0) tc_mbar_arrive(bar_loaded);
          continue;
        }
        if (tc_elect()) {
          if (qs > 0 && !tc_mbar_wait(bar_qfree, (qs - 1) & 1)) timed_out = true;
          if (!timed_out) {
            tc_mbar_expect_tx(bar_q, ((w.n[0] > 0) + (w.n[1] > 0)) * p.tokens * p.pack * DP * 2);
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (w.n[t] > 0)
                for (int i = 0; i < DP / 64; ++i)
                  pa_tma_3d(sbase + t * C::kTileBytes + i * SUB, &qmap, 64 * i, w.head[t], w.q0 + w.row[t], bar_q);
          }
          for (int i2 = 0; i2 < 2 * nmax && !timed_out; ++i2) {
            const int it = it0 + i2, s = it % C::kStages;
            if (!tc_mbar_wait(bar_empty + 8 * s, ((it / C::kStages) & 1) ^ 1)) {
              timed_out = true;
              break;
            }
            tc_mbar_expect_tx(bar_full + 8 * s, C::kTileBytes);
            for (int i = 0; i < DP / 64; ++i)
              pa_tma_3d(sbase + C::kOffKv + s * C::kTileBytes + i * SUB, (i2 & 1) ? &vmap : &kmap, 64 * i, w.kvh,
                        w.k0 + (i2 >> 1) * kKeys, bar_full + 8 * s);
          }
        }
        timed_out = __any_sync(~0u, timed_out);
        if (lane == 0) tc_mbar_arrive(bar_loaded);
        it0 += 2 * nmax;
        ++qs;
        if (dirty(w, nmax)) {                   // the last tile of V reaches into another request: clear those rows
          const int it = it0 - 1, s = it % C::kStages;
          if (!timed_out && !tc_mbar_wait(bar_full + 8 * s, (it / C::kStages) & 1)) timed_out = true;
          if (!timed_out) {
            const int r0 = w.nk - (nmax - 1) * kKeys;           // first row of another request
            const uint32_t tile = sbase + C::kOffKv + s * C::kTileBytes;
            for (int i = lane; i < (kKeys - r0) * 8 * (DP / 64); i += 32) {
              const int sub = i / ((kKeys - r0) * 8), x = i - sub * ((kKeys - r0) * 8);
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + sub * SUB + r0 * 128 + x * 16), "r"(0) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          timed_out = __any_sync(~0u, timed_out);
          if (lane == 0) tc_mbar_arrive(bar_clean + 8 * (cleans % kCleans));
          ++cleans;
        }
      }
      // given up: what has been asked for arrives before the CTA leaves (each tile's wait is bounded, too)
      if (timed_out && lane == 0)
        for (int it = max(it0 - C::kStages, 0); it < it0; ++it) tc_mbar_wait(bar_full + 8 * (it % C::kStages), (it / C::kStages) & 1);
    } else if (warp == kMmaWarp) {
      // ------------------------------------------------------------------ MMAs
      if (tc_elect()) {
        constexpr uint32_t kType = BF16 ? (1u << 7) | (1u << 10) : 0u;
        const uint32_t idesc_s = (1u << 4) | kType | ((uint32_t)(kKeys >> 3) << 17) | (8u << 24);
        const int nv = (p.dv + 15) / 16 * 16, ks = (p.dk + 15) / 16;
        const uint32_t idesc_o = (1u << 4) | kType | (1u << 16) | ((uint32_t)(nv >> 3) << 17) | (8u << 24);
        auto wait = [&](uint32_t bar, uint32_t parity) {
          if (!timed_out && !tc_mbar_wait(bar, parity)) timed_out = true;
          tc_fence_after();
        };
        auto scores = [&](int t, int it) {      // S_t = Q_t K^T with the tile of item it
          const uint32_t kt = sbase + C::kOffKv + (it % C::kStages) * C::kTileBytes, qt = sbase + t * C::kTileBytes;
          if (!timed_out)
            for (int s = 0; s < ks; ++s)
              pa_mma_ss(tmem + t * 128, tc_smem_desc(qt + (s >> 2) * SUB) + 2 * (s & 3),
                        tc_smem_desc(kt + (s >> 2) * SUB) + 2 * (s & 3), idesc_s, s > 0);
          tc_commit(bar_s + 8 * t);
        };
        auto values = [&](int t, int it, uint32_t acc, uint32_t parity) {        // O_t (+)= P_t V, half by half as P arrives
          const uint32_t vt = sbase + C::kOffKv + (it % C::kStages) * C::kTileBytes;
          // MN-major, 128-byte swizzle: 64-channel sub-tiles SUB bytes apart, groups of 8 keys 1024 bytes apart
          const uint64_t vd = (uint64_t)((vt & 0x3FFFFu) >> 4) | ((uint64_t)(SUB >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            wait(bar_p + 16 * t + 8 * h, parity);
            if (!timed_out)
#pragma unroll
              for (int s = 4 * h; s < 4 * h + 4; ++s)
                pa_mma_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * s, vd + 128 * s, idesc_o, s > 0 ? 1u : acc);
          }
          tc_commit(bar_o + 8 * t);
        };
        PaItem w;
        int it0 = 0, qs = 0, cleans = 0, steps[2] = {0, 0}, outs[2] = {0, 0};     // tiles, items, .. so far; steps and results of a unit
        for (int k = 0; item(k, w, false); ++k) {
          tc_mbar_arrive(bar_taken + 8 * (k & 1));
          const int nmax = max(w.n[0], w.n[1]);
          if (nmax == 0) continue;
          const bool unclean = dirty(w, nmax);
          wait(bar_q, qs & 1);
          wait(bar_full + 8 * (it0 % C::kStages), (it0 / C::kStages) & 1);
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (w.n[t] > 0) scores(t, it0);
          tc_commit(bar_empty + 8 * (it0 % C::kStages));
          if (nmax == 1) tc_commit(bar_qfree);
          for (int j = 0; j < nmax; ++j) {
            const int iv = it0 + 2 * j + 1, ik = iv + 1, sv = iv % C::kStages, sk = ik % C::kStages;
            wait(bar_full + 8 * sv, (iv / C::kStages) & 1);
            if (j + 1 < nmax) wait(bar_full + 8 * sk, (ik / C::kStages) & 1);
            else if (unclean) wait(bar_clean + 8 * (cleans % kCleans), (cleans / kCleans) & 1);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (j < w.n[t]) {
                // the first values of an item overwrite the unit's result before it: that has to have been read
                if (j == 0 && outs[t] > 0) wait(bar_ofree + 8 * t, (outs[t] - 1) & 1);
                values(t, iv, j > 0, (steps[t] + j) & 1);
              }
              if (t == 1) tc_commit(bar_empty + 8 * sv);
              if (j + 1 < w.n[t]) scores(t, ik);
            }
            if (j + 1 < nmax) tc_commit(bar_empty + 8 * sk);
            if (j + 2 == nmax) tc_commit(bar_qfree);            // the item's last Q K^T
          }
          it0 += 2 * nmax;
          ++qs;
          cleans += unclean;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            steps[t] += w.n[t];
            outs[t] += w.n[t] > 0;
          }
        }
      }
    }
    } else {
      // ------------------------------------------------------------------ softmax, one query row a thread
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
      const int t = warp >> 2;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + t * 128 + lanes, to = tmem + 256 + t * 128 + lanes;
      const float f = p.scale_log2;
      const int r = (warp & 3) * 32 + lane, my_token = r / p.pack, my_head = r - my_token * p.pack;
      const int tokens = p.tokens;
      PaItem w;
      int steps = 0;                            // of this unit in the items before
      for (int k = 0; item(k, w, true); ++k) {
      __syncwarp();
      if (lane == 0) tc_mbar_arrive(bar_taken + 8 * (k & 1));
      const int nt = t ? w.n[1] : w.n[0], row0 = t ? w.row[1] : w.row[0], head = t ? w.head[1] : w.head[0];
      const int nq = w.nq, nk = w.nk, shift = nk - nq, i = row0 + my_token;
      const int limit = p.causal ? min(nk, max(i + 1 + shift, 0)) : nk;
      const int full = p.causal ? min(nk, max(row0 + 1 + shift, 0)) : nk;       // keys that every row of the unit sees
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nt; ++j) {
        if (!timed_out && !tc_mbar_wait(bar_s + 8 * t, (steps + j) & 1)) timed_out = true;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) pa_ld32(ts + 32 * c, s + 32 * c);
        pa_wait_ld();
        const bool masked = (j + 1) * kKeys > full;
        if (masked) {
          const int left = limit - j * kKeys;
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c < left ? s[c] : -INFINITY;
        }
        float top4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < 124; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) top4[e] = pa_max3(top4[e], s[c + e], s[c + 4 + e]);
        float top = pa_max3(pa_max3(top4[0], top4[1], top4[2]), pa_max3(top4[3], s[124], s[125]), pa_max3(s[126], s[127], s[127]));
        top = i < nq && my_token < tokens ? top * f : -INFINITY;        // rows of another request, or of none, have no say in when m is raised
        if (top != top) m = top;                // a NaN among the scores: all of the row is
        if (__any_sync(~0u, top > m + 8.f)) {
          const float mn = fmaxf(m, top);
          const float down = m == m ? (mn == -INFINITY ? 1.f : pa_exp2(m - mn)) : m;
          m = m == m ? mn : m;
          l *= down;
          if (j > 0) {
            if (!timed_out && !tc_mbar_wait(bar_o + 8 * t, (steps + j - 1) & 1)) timed_out = true;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              float o[32];
              pa_ld32(to + c, o);
              pa_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= down;
              pa_st32(to + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        const uint64_t ff = two(f, f), nb = two(-base, -base);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {           // P = 2^(f S - m), 32 columns at a time
          uint32_t y[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 x = split2(fma2(two(s[32 * q + 2 * c], s[32 * q + 2 * c + 1]), ff, nb));
            const float2 e = make_float2(pa_exp2(x.x), pa_exp2(x.y));
            sum[c & 1] = add2(sum[c & 1], two(e.x, e.y));
            y[c] = pa_pack<BF16>(e.x, e.y);
          }
          pa_st16(ts + 16 * q, y);
          if (q & 1) {
            pa_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(bar_p + 16 * t + 8 * (q >> 1));
          }
        }
        const float2 s0 = split2(sum[0]), s1 = split2(sum[1]);
        l += (s0.x + s0.y) + (s1.x + s1.y);
      }
      // ---- O / l
      if (head >= 0) {
        if (nt > 0) {
          if (!timed_out && !tc_mbar_wait(bar_o + 8 * t, (steps + nt - 1) & 1)) timed_out = true;
          tc_fence_after();
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        unsigned char* dst = p.out + ((size_t)(w.q0 + i) * p.heads + head + my_head) * p.dv * 2;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          float o[32];
          if (nt > 0) {
            pa_ld32(to + c, o);
            pa_wait_ld();
            if (c + 32 == DP) {                 // O may be overwritten
              tc_fence_before();
              __syncwarp();
              if (lane == 0) tc_mbar_arrive(bar_ofree + 8 * t);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (i < nq && my_token < tokens && !timed_out) {
            uint32_t x[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = l == 0.f ? 0u : pa_pack<BF16>(o[2 * e] * inv, o[2 * e + 1] * inv);
#pragma unroll
            for (int v = 0; v < 2; ++v) {       // a store instruction touches 32 rows: the fewer, the better
              unsigned char* at = dst + (c + 16 * v) * 2;
              if (p.wide) {
                if (c + 16 * v < p.dv) pa_store32(at, x + 8 * v);
              } else {
                if (c + 16 * v < p.dv) *reinterpret_cast<uint4*>(at) = make_uint4(x[8 * v], x[8 * v + 1], x[8 * v + 2], x[8 * v + 3]);
                if (c + 16 * v + 8 < p.dv) *reinterpret_cast<uint4*>(at + 16) = make_uint4(x[8 * v + 4], x[8 * v + 5], x[8 * v + 6], x[8 * v + 7]);
              }
            }
          }
        }
      }
      steps += nt;
      }
  }
  if (timed_out && p.status_word) atomicOr(p.status_word, UNIQL_STATUS_WAIT_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// rows [tokens, heads, d] as a 3-D tensor, boxes of 64 channels x box_heads x box_tokens; what lies outside reads as zero
static int pa_map(CUtensorMap* map, const void* x, int64_t tokens, int64_t heads, int64_t d, int64_t token_stride,
                  int64_t head_stride, bool bf16, int box_heads = 1, int box_tokens = 128) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return cuda_fail(cudaErrorNotSupported);
  cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, estr[3] = {1, 1, 1};
  if (enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(x), dims, strides,
          box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cuda_fail(cudaErrorInvalidValue);
  return UNIQL_OK;
}

template <int DP, bool BF16>
static int pa_launch(const PaParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, unsigned ctas, cudaStream_t stream) {
  static thread_local bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    UNIQL_CUDA_TRY(cudaFuncSetAttribute(prompt_attention_kernel<DP, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, pa::Cfg<DP>::kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(pa::kThreads);
  cfg.dynamicSmemBytes = pa::Cfg<DP>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  UNIQL_CUDA_TRY(cudaLaunchKernelEx(&cfg, prompt_attention_kernel<DP, BF16>, p, q, k, v));
  return UNIQL_OK;
}

}  // namespace uniql

extern "C" int uniql_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                      int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                      int64_t v_head_stride, const int32_t* cu_q, const int32_t* cu_k, int64_t batch,
                                      int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv,
                                      float softmax_scale, int causal, int dtype, void* out, int* status_word, void* stream) {
  using namespace uniql;
  if (batch < 0 || total_q < 0 || total_k < 0 || heads <= 0 || kv_heads <= 0 || dk <= 0 || dv <= 0) return UNIQL_EINVAL;
  if (dtype != UNIQL_F16 && dtype != UNIQL_BF16) return UNIQL_EDTYPE;
  if (dk % 8 || dv % 8 || dk > 128 || dv > 128 || heads % kv_heads || heads > 16384 || kv_heads > 1024) return UNIQL_ESHAPE;
  // 2^26 keys are 2^19 tiles, 0.8 s of one item: well inside the bound of every wait
  if (batch > UNIQL_KV_MAX_BATCH || total_q > kMaxTokens || total_k > (int64_t)1 << 26) return UNIQL_ESHAPE;
  if (!(softmax_scale > 0.f) || softmax_scale > 1e30f) return UNIQL_EINVAL;
  if ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return UNIQL_EINVAL;
  if (q_token_stride < 0 || q_head_stride < 0 || k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
    return UNIQL_EINVAL;
  if (total_q == 0) return UNIQL_OK;
  if (!q || !out || !aligned16(q) || !aligned16(out)) return UNIQL_EINVAL;
  if (total_k > 0 && (!k || !v || !aligned16(k) || !aligned16(v))) return UNIQL_EINVAL;
  if (batch > 0 && (!cu_q || !cu_k)) return UNIQL_EINVAL;
  PaParams p;
  p.cu_q = cu_q; p.cu_k = cu_k; p.out = (unsigned char*)out; p.status_word = status_word;
  p.batch = (int)batch; p.total_q = (int)total_q; p.total_k = (int)total_k; p.heads = (int)heads; p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads); p.dk = (int)dk; p.dv = (int)dv; p.causal = causal != 0;
  p.scale_log2 = softmax_scale * 1.44269504088896340736f;
  const bool bf16 = dtype == UNIQL_BF16;
  // Rows of a unit: 128 tokens of one query head, or, where that leaves fewer units, fewer tokens of the whole group, a token's
  // heads side by side (a short request, or the end of a long one, fills its last row block better; us apart / packed: 64
  // requests of one token, 28 heads over 4 kv heads 45.8 / 17.7, 32 of 400 tokens 111 / 93, 16 mixed prompts 481 / 453, one of
  // 16384 the same).  At most this many units: every request rounds its row blocks up.
  const int64_t sms = device_info().sm_count, some = batch < total_q ? batch : total_q;
  p.pack = 1;
  if (p.group > 1 && p.group <= pa::kRows) {
    const int64_t apart = (total_q / pa::kRows + some) * p.group, packed = total_q / (pa::kRows / p.group) + some;
    if (packed * 64 <= apart * 63) p.pack = p.group;
  }
  p.tokens = pa::kRows / p.pack; p.parts = p.group / p.pack;
  CUtensorMap qm, km, vm;
  int st = pa_map(&qm, q, total_q, heads, dk, q_token_stride, q_head_stride, bf16, p.pack, p.tokens);
  // without keys no tile of K or V is ever loaded: the maps only have to be valid
  if (st == UNIQL_OK) st = total_k ? pa_map(&km, k, total_k, kv_heads, dk, k_token_stride, k_head_stride, bf16) : (km = qm, UNIQL_OK);
  if (st == UNIQL_OK) st = total_k ? pa_map(&vm, v, total_k, kv_heads, dv, v_token_stride, v_head_stride, bf16) : (vm = qm, UNIQL_OK);
  if (st != UNIQL_OK) return st;
  const int64_t blocks = total_q / p.tokens + some;
  // two units share an SM and their keys only when there are not SMs enough for one each
  p.units = blocks * p.parts * kv_heads <= sms ? 1 : 2;
  p.wide = dv % 16 == 0 && !(reinterpret_cast<uintptr_t>(out) & 31);
  const int64_t items = p.units == 1 ? blocks * p.parts : (blocks * p.parts + 1) / 2 + batch;
  int64_t ctas = items * kv_heads;
  if (ctas < sms) ctas = total_q < sms ? (ctas > total_q ? ctas : total_q) : sms;       // rows that nobody owns are cleared by all
  if (ctas > ((int64_t)1 << 31) - 1) return UNIQL_ESHAPE;
  cudaStream_t s = (cudaStream_t)stream;
  if (dk > 64 || dv > 64)
    return bf16 ? pa_launch<128, true>(p, qm, km, vm, (unsigned)ctas, s) : pa_launch<128, false>(p, qm, km, vm, (unsigned)ctas, s);
  return bf16 ? pa_launch<64, true>(p, qm, km, vm, (unsigned)ctas, s) : pa_launch<64, false>(p, qm, km, vm, (unsigned)ctas, s);
}
