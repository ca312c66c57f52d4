// Attention of one query token per request over a paged KV cache held in 4 bits.  Layout and rules: include/uniql_b200.h.
//
// Mathematics.  With a cached row k_t = z + s c and m = z + 8 s the score is  x_t = f (s (q . (c - 8)) + m sum(q)),  f =
// softmax_scale log2(e).  q . (c - 8) is integer arithmetic on the tensor cores: four codes are the bytes of one AND, q is a fixed-point
// number that is off by at most 2^-19 of its largest channel, split into three signed base-128 digits, and mma.sync m16n8k32 (u8 x s8)
// sums digit times code for each, exactly.  A packed word costs three instructions, all a half-rate pipe's, against five of that pipe
// and four of the other one as two fp16 pairs: what bounds the arithmetic is that pipe (LOP3, PRMT, shifts: two cycles each).  (As
// e4m3 products, where a code is its own subnormal number, the kernel was no faster.)  Scale and zero enter once per token in fp32.
// The value side folds its scale into the exponent: with y_t = x_t + log2 s'_t, M a running bound of y and w_t = 2^(y_t - M),
//     out = (sum w_t (c'_t - 8) + sum (w_t / s'_t) m'_t) / sum (w_t / s'_t),
// so that of the second product w alone is rounded (fp16: by 2^-11 of itself, by 2^-25 below 6e-5; it is at most 2^8, see below), next to
// exact fp16 codes, whatever the magnitude of the values.  M is raised, and the sums rescaled, only when some y exceeds it by more
// than 8.
//
// What has fewer than 32 bits, and why: q's 20 bits in fixed point (small channels beside an outlier lose theirs; a row whose largest
// channel is below 2^-107 counts as zeros), because the integer products take three digits; and w, because the second product would
// cost twice as much with what fp16 leaves of it as another operand.  The sums of w are taken before it is rounded, and all sums, the
// bound and the parts are fp32.  Error against 64 bits beside that of fp32 arithmetic, whose results are rounded alike: 1.0 to 1.2
// times up to a few thousand tokens, 1.4 times (3.0e-4 of the result) at 131072.
//
// Layout of the products.  Tokens are the 16-row operand of the first product (a lane's packed words of two tokens are its
// fragment; which channel sits at which k index is free, so long as the query fragments follow), query heads its eight
// columns.  The weights w cross to the second product by 8 x 8 transposes (movmatrix); there channels are the rows and the
// tokens of a lane meet pairwise: byte permutes join the same nibbles of two tokens.  So the 4-bit words go from shared memory
// to the tensor cores in registers.
//
// Bound: HBM, (dk + dv) / 2 + 8 bytes per token and kv head, and close behind it the arithmetic: at 8 x 131072 tokens, 8 kv heads
// (174 us at the measured copy rate), the loads alone take 180 us, the arithmetic alone 195 (as fp16 products), both 225 in a short
// burst and 245 to 260 back to back, where the power limit lowers the clock.  Each
// warp keeps a ring of kStages steps of 32 tokens in flight with cp.async.
//
// Split: lengths are read on the device, and every CTA works out the same cut from them.  A step is 32 tokens of one request and kv
// head, a list the steps of one request and head.
//  - Little work (below kShort steps a CTA): lists are cut into equal parts of about 8 to 32 steps, one a CTA, as long as all
//    are resident at once.  A list that is one part is finished where it is read: joining parts costs 3.5 us of dependent trips
//    to L2, as much as 32 steps.  (us, parts / ranges: 250 tokens of 1 request 8.4 / 10.1, of 32 requests 11.8 / 13.9, 4000
//    tokens of 1 request 13.0 / 18.2, 16000 of 1 20.3 / 27.0; 1000 of 1 11.1 / 11.3.)
//  - More: the steps form one long list, cut into equal ranges, one per CTA.  Every list begins with kOpen places that stand for
//    what a CTA pays to open it (queries, first loads, the join), so that ranges with several lists hold fewer steps (64 ragged
//    requests: 57 us without, 50 with 16).
// A CTA that has only a part of a list stores an fp32 partial (sums, M), and the last CTA of that list to arrive joins the parts
// in order: deterministic.
#include "common.cuh"
#include "kv_cache.cuh"
#include "tma.cuh"

#include <type_traits>

namespace uniql {

namespace kva {
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kStep = 32;                       // tokens of a step: one warp, one turn of its ring
constexpr int kOpen = 16;                       // what opening a list costs a CTA, in steps: places of the list that hold no tokens
constexpr int kShort = 24;                      // below so many steps a CTA lists are cut into whole parts
// steps of a part, and how many parts a list may have: joining takes longer the more there are
__host__ __device__ constexpr int part_steps(int k) { return k == 0 ? 8 : k == 1 ? 12 : k == 2 ? 24 : 32; }
__host__ __device__ constexpr int most_parts(int k) { return k < 2 ? 12 : 24; }
constexpr float kFloor = -1e30f;                // M before the first token
constexpr int kMaxCtas = 2048;
constexpr int per_sm(int nt) { return nt == 1 ? 3 : 2; }        // resident CTAs (NT 1: 237 us with 3, 245 with 2, 251 with 4 at 8 x 131072)
}  // namespace kva

struct KvaParams {
  const unsigned char* q;
  int64_t q_bs, q_hs;                           // elements
  const unsigned char* codes;
  const unsigned char* scales;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lens;
  unsigned char* out;
  float* part;                                  // [2 * ctas][8 NT][DP + 4]
  int* tickets;                                 // [ctas], zero
  int* status_word;
  int batch, heads, kv_heads, group, hgroups;   // group: query heads of a kv head; hgroups: launches of 8 NT of them
  int max_blocks, num_pages, page_shift, dk, dv, bf16, q_vec;     // q_vec: rows of q are 16-byte aligned
  float scale_log2;
};

__device__ __forceinline__ void kva_cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t kva_lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float kva_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kva_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float kva_load(const unsigned char* p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void kva_store(unsigned char* p, int64_t i, int bf16, float v) {
  if (bf16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ void kva_mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kva_lds2(uint32_t a, uint64_t& x, uint64_t& y) {
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(x), "=l"(y) : "r"(a) : "memory");
}
__device__ __forceinline__ float kva_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kva_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The token (of 16) that sits at row / k index r of the products: k = 2c, 2c + 1, 2c + 8, 2c + 9 are tokens c, 7 - c, 8 + c
// and 15 - c.  With it, and the 16-byte chunks of 64-byte rows swapped in pairs by bit 1 of the token, both the rows (four lanes
// a row) and the columns (eight lanes a row, four tokens) are read from shared memory without bank conflicts.
__device__ __forceinline__ int kva_token(int r) { return (r & 8) + ((r & 1) ? 7 - ((r & 7) >> 1) : ((r & 7) >> 1)); }

template <int DP>
struct KvaVec {                                 // a lane's channels of a part
  using T = float4;
};
template <>
struct KvaVec<64> {
  using T = float2;
};

// The parts of a list, from CTAs c0 .. c1, into `rows` rows of the output from `row0` on.  A warp per head: lanes hold the parts' M and
// L, 32 at a time, then every lane adds up its channels part by part; the first parts' sums are on their way meanwhile (two: with
// eight the registers of the loop spill, 222 -> 227 us at 8 x 131072 tokens).
template <int DP, int H>
__device__ __forceinline__ void kva_join_parts(const KvaParams& p, int64_t row0, int rows, int c0, int c1) {
  using namespace kva;
  using Vec = typename KvaVec<DP>::T;
  constexpr int PSTR = DP + 4, AHEAD = 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int h = warp; h < rows; h += kWarps) {
    auto part = [&](int k) { return p.part + ((size_t)(2 * k + (k == c0)) * H + h) * PSTR; };
    auto sums = [&](int k) { return __ldcg(reinterpret_cast<const Vec*>(part(k) + lane * (DP / 32))); };
    Vec ahead[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (c0 + k <= c1) ahead[k] = sums(c0 + k);
    float m = kFloor, lw = 0.f;
    if (c0 + lane <= c1) {
      m = __ldcg(part(c0 + lane) + DP);
      lw = __ldcg(part(c0 + lane) + DP + 1);
    }
    float top = m;
    for (int k = c0 + 32 + lane; k <= c1; k += 32) top = fmaxf(top, __ldcg(part(k) + DP));
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
    float acc[DP / 32], l = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) acc[e] = 0.f;
    auto add = [&](float wk, const Vec& v) {
      const float* x = reinterpret_cast<const float*>(&v);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) acc[e] = fmaf(wk, x[e], acc[e]);
    };
    for (int k0 = c0; k0 <= c1; k0 += 32) {
      const int n = min(32, c1 - k0 + 1);
      if (k0 > c0 && lane < n) {
        m = __ldcg(part(k0 + lane) + DP);
        lw = __ldcg(part(k0 + lane) + DP + 1);
      }
      const float w = lane < n ? kva_exp2(m - top) : 0.f;
      float sum = lane < n ? w * lw : 0.f;
#pragma unroll
      for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(~0u, sum, s);
      l += sum;
      int k = 0;
      if (k0 == c0) {
#pragma unroll
        for (; k < AHEAD; ++k)
          if (k < n) add(__shfl_sync(~0u, w, k), ahead[k]);
      }
#pragma unroll 4
      for (; k < n; ++k) add(__shfl_sync(~0u, w, k), sums(k0 + k));
    }
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) {
      const int d = lane * (DP / 32) + e;
      if (d < p.dv) kva_store(p.out, (row0 + h) * p.dv + d, p.bf16, l == 0.f ? 0.f : acc[e] / l);
    }
  }
}

template <int DP, int NT, bool PAGE16>
__global__ void __launch_bounds__(kva::kThreads, kva::per_sm(NT)) kv4_attention_kernel(const __grid_constant__ KvaParams p) {
  using namespace kva;
  constexpr int ROWB = DP / 2;                  // bytes of a packed row
  constexpr int CODEB = 16 * ROWB;              // packed rows of 16 tokens, K or V
  constexpr int OFF_SC = 4 * CODEB;             // of a stage: K codes (two halves of 16 tokens), V codes, then 128 bytes of scales a half
  constexpr int STAGEB = OFF_SC + 256;
  constexpr int RINGB = kStages * STAGEB, WARPB = RINGB + kStep * 40;
  constexpr int H = 8 * NT, MT = DP / 16, KS = DP / 32;
  constexpr int PSTR = DP + 4;                  // floats of one head's partial: sums, M, L
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long s_wide[kWarps];
  __shared__ unsigned s_count[kWarps][6];
  __shared__ float s_m[kWarps][H], s_l[kWarps][H], s_z[kWarps][H];
  __shared__ int s_find;
  __shared__ long long s_before;
  __shared__ int s_last;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int cap = min((int64_t)p.max_blocks << p.page_shift, (int64_t)kMaxTokens);
  const int lists = p.kv_heads * p.hgroups;     // lists of a request
  auto length = [&](int b) { return min(max(p.lens[b], 0), cap); };

  // ---- how the lists are cut
  int unit = 0;                                 // steps of a part; 0: the ranges of one long list
  auto cut = [&](unsigned work, unsigned longest, const unsigned (&parts)[4]) {
    if ((long long)work * lists >= (long long)kShort * gridDim.x) return;
#pragma unroll
    for (int k = 3; k >= 0; --k)
      if ((long long)parts[k] * lists <= gridDim.x && longest <= part_steps(k) * most_parts(k)) unit = part_steps(k);
    // lists that are joined anyway: a step a warp
    if (unit == part_steps(0) && longest > part_steps(0) && longest <= kWarps * most_parts(0) && 2ll * parts[0] * lists <= gridDim.x) unit = kWarps;
  };
  // a list's places: its parts, or its steps and what stands for the opening
  auto places = [&](int len) {
    const int steps = (len + kStep - 1) / kStep;
    return len <= 0 ? 0 : unit ? (steps + unit - 1) / unit : steps + kOpen;
  };
  long long begin = 0, end = 0, N;              // this CTA's range of the list of all places
  long long ctas;
  auto range = [&](long long total) {
    N = total * lists;                          // below 2^48, times the CTAs below 2^59
    ctas = min((long long)gridDim.x, N);
    if (blockIdx.x >= ctas) return;
    begin = N * blockIdx.x / ctas;              // parts: one each
    end = N * (blockIdx.x + 1) / ctas;
  };
  int b;
  long long req_begin;
  if (p.batch <= 32) {                          // every warp by itself, a request a lane: no barrier on the way to the first load
    const int len = lane < p.batch ? length(lane) : 0;
    const unsigned steps = (unsigned)(len + kStep - 1) / kStep, few = min(steps, 1u << 14);
    unsigned parts[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) parts[k] = __reduce_add_sync(~0u, (few + part_steps(k) - 1) / part_steps(k));
    cut(__reduce_add_sync(~0u, few), __reduce_max_sync(~0u, few), parts);
    const unsigned mine = places(len);          // below 2^24, 32 of them below 2^29
    unsigned incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    range(__shfl_sync(~0u, incl, 31));
    const unsigned has = __ballot_sync(~0u, mine && (long long)(incl - mine) * lists <= begin && begin < (long long)incl * lists);
    b = has ? __ffs(has) - 1 : 0;
    req_begin = (long long)__shfl_sync(~0u, incl - mine, b) * lists;
  } else {
    const int per = (p.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    unsigned work = 0, longest = 0, parts[4] = {0, 0, 0, 0};    // what is too large for the whole cut anyway is counted short
    for (int i = b0; i < b1; ++i) {
      const unsigned steps = min((unsigned)(length(i) + kStep - 1) / kStep, 1u << 14);
      work += steps;
      longest = max(longest, steps);
#pragma unroll
      for (int k = 0; k < 4; ++k) parts[k] += (steps + part_steps(k) - 1) / part_steps(k);
    }
    work = __reduce_add_sync(~0u, work);
    longest = __reduce_max_sync(~0u, longest);
#pragma unroll
    for (int k = 0; k < 4; ++k) parts[k] = __reduce_add_sync(~0u, parts[k]);
    if (lane == 0) {
      s_count[warp][0] = work;
      s_count[warp][1] = longest;
#pragma unroll
      for (int k = 0; k < 4; ++k) s_count[warp][2 + k] = parts[k];
    }
    __syncthreads();
    work = longest = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) parts[k] = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      work += s_count[w][0];
      longest = max(longest, s_count[w][1]);
#pragma unroll
      for (int k = 0; k < 4; ++k) parts[k] += s_count[w][2 + k];
    }
    cut(work, longest, parts);
    long long mine = 0;
    for (int i = b0; i < b1; ++i) mine += places(length(i));
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_wide[warp] = incl;
    __syncthreads();
    long long total = 0, before = incl - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_wide[w];
      total += s_wide[w];
    }
    range(total);
    if (mine && before * lists <= begin && begin < (before + mine) * lists) {
      long long at = before;
      for (int i = b0; i < b1; ++i) {
        const int t = places(length(i));
        if (begin < (at + t) * lists) {
          s_find = i;
          s_before = at * lists;
          break;
        }
        at += t;
      }
    }
    __syncthreads();
    b = s_find;                                 // of a CTA with places
    req_begin = s_before;
  }
  // idle rows of the batch
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (length(b) == 0)
      for (int i = tid; i < p.heads * p.dv; i += kThreads) kva_store(p.out, (int64_t)b * p.heads * p.dv + i, p.bf16, 0.f);
  if (begin == end) return;

  const uint32_t ring = smem_addr(smem) + warp * WARPB, meta = ring + RINGB;
  const int tok_a = kva_token(g);               // rows g and g + 8 of the first product: tokens tok_a and 8 + tok_a
  const int pmask = (1 << p.page_shift) - 1;
  // bytes of a page (at most 2^25) and from its K to its V
  const uint32_t page_codes = (uint32_t)(2 * p.kv_heads * ROWB) << p.page_shift, v_codes = page_codes / 2;
  const uint32_t page_scales = (uint32_t)(8 * p.kv_heads) << p.page_shift;
  // where a lane's 16-byte chunk of packed words goes: chunk of token t = lane / 4 moves to chunk ^ (t & 2)
  const uint32_t lane_dst = DP == 128 ? (lane * 16) ^ ((lane & 8) << 2) : lane * 16;
  bool bad_page = false;

  for (long long cur = begin; cur < end;) {
    int len = length(b);
    int size = places(len);
    while (cur >= req_begin + (long long)size * lists) {        // next request that has tokens
      req_begin += (long long)size * lists;
      ++b;
      len = length(b);
      size = places(len);
    }
    const int list = (int)((cur - req_begin) / size);
    const long long list_begin = req_begin + (long long)list * size;
    const int at = (int)(cur - list_begin), steps = (len + kStep - 1) / kStep;
    int t0, t1;                                                 // steps of this list
    if (unit) {
      t0 = steps * at / size;
      t1 = steps * (at + 1) / size;
      ++cur;
    } else {
      t0 = max(at - kOpen, 0);
      t1 = (int)min((long long)size, end - list_begin) - kOpen;
      cur = list_begin + min((long long)size, end - list_begin);
      if (t1 <= t0) continue;                                   // only places that stand for the opening
    }
    const int kvh = list / p.hgroups, hg = list - kvh * p.hgroups;
    const int head0 = kvh * p.group + hg * H;                   // first query head of this list
    const int nh = min(H, p.group - hg * H);

    // ---- producer: 32 tokens into a ring slot.  A page of 16 holds half a step; larger ones hold whole steps
    const int first = t0 + warp;                                // this warp's steps: first, first + kWarps, .. < t1
    const int32_t* trow = p.table + (size_t)b * p.ld_table;
    const unsigned char* kbase = p.codes + (((int64_t)kvh * ROWB) << p.page_shift) + lane * 16;
    const unsigned char* sbase = p.scales + (((int64_t)kvh * 4) << p.page_shift) + ((lane & 4) ? page_scales / 2 : 0) + (lane & 3) * 16;
    const int last_block = (len - 1) >> p.page_shift;
    int page0 = 0, page1 = 0;                                   // of the step that is produced next
    auto look = [&](int st) {
      page0 = trow[st * kStep >> p.page_shift];
      if (PAGE16) page1 = trow[min(2 * st + 1, last_block)];
    };
    if (first < t1) look(first);

    // ---- this list's queries, while the first page number is on its way
    float v[NT][DP / 4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const int64_t base = (int64_t)b * p.q_bs + (int64_t)(head0 + h) * p.q_hs;
#pragma unroll
      for (int i = 0; i < DP / 4; i += 8) {
        const int d = c * (DP / 4) + i;
        if (h < nh && d < p.dk) {
          if (p.q_vec) {
            const uint4 w = *reinterpret_cast<const uint4*>(p.q + 2 * (base + d));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 t = p.bf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[e]))
                                      : __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
              v[nt][i + 2 * e] = t.x;
              v[nt][i + 2 * e + 1] = t.y;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[nt][i + e] = kva_load(p.q, base + d + e, p.bf16);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[nt][i + e] = 0.f;
        }
      }
    }

    auto produce = [&](int st, uint32_t dst) {
      if (st < t1) {
        int pg0 = page0, pg1 = PAGE16 ? page1 : page0;
        if (st + kWarps < t1) look(st + kWarps);
        const bool ok0 = (unsigned)pg0 < (unsigned)p.num_pages, ok1 = (unsigned)pg1 < (unsigned)p.num_pages;
        if (!ok0) pg0 = 0;                                      // an absent page: copies of no bytes, zeros in the ring
        if (!ok1) pg1 = 0;
        bad_page |= !(ok0 && ok1);
        const uint32_t at = (st * kStep) & pmask;
        const unsigned char* src0 = kbase + (uint64_t)pg0 * page_codes + at * ROWB;
        // the second half is the next 16 rows, or the first 16 of the next page
        const unsigned char* src1 = PAGE16 ? kbase + (uint64_t)pg1 * page_codes : src0 + CODEB;
        const uint32_t d = dst + lane_dst;
#pragma unroll
        for (int i = 0; i < CODEB / 512; ++i) {
          kva_cp16(d + 512 * i, src0 + 512 * i, ok0);
          kva_cp16(d + 512 * i + CODEB, src1 + 512 * i, ok1);
          kva_cp16(d + 512 * i + 2 * CODEB, src0 + v_codes + 512 * i, ok0);
          kva_cp16(d + 512 * i + 3 * CODEB, src1 + v_codes + 512 * i, ok1);
        }
        if (lane < 16) {                                        // 64 bytes of K scales, 64 of V scales, twice
          const uint32_t row = PAGE16 ? 0u : at + (lane & 8) * 2;
          kva_cp16(dst + OFF_SC + lane * 16, sbase + (uint64_t)(lane < 8 ? pg0 : pg1) * page_scales + row * 4, lane < 8 ? ok0 : ok1);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) produce(first + i * kWarps, ring + i * STAGEB);

    // ---- query digits: k index 4c + e of step i is channel 8 (KS c + i) + 2e, k index 16 + 4c + e the one behind it
    uint32_t qf[NT][3][KS][2];
    uint64_t f[NT], fq[NT];                     // pairs of heads 8 nt + 2c, 2c + 1: f times the unit of the digits, f sum(q)
    int init[NT][2];                            // -8 times the digits' value, summed
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 4; ++i) {
        top = fmaxf(top, fabsf(v[nt][i]));
        sum += v[nt][i];
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        sum += __shfl_xor_sync(~0u, sum, o);
      }
      // down = 2^(18 - e), up = 2^(e - 18) for 2^e <= top < 2^(e + 1); a row below 2^-107 counts as zeros, and one that is not
      // finite (sum - sum is NaN then, or top is infinite) makes its scores NaN
      const int eb = (__float_as_int(top) >> 23) & 255;
      const bool live = eb >= 20 && eb < 255;
      const float down = live ? __int_as_float((272 - eb) << 23) : 0.f, up = live ? __int_as_float((eb - 18) << 23) : 0.f;
      int digits[3] = {0, 0, 0};                // their sums
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          uint32_t w[3] = {0, 0, 0};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // q down rounded to an integer in the low bits of a float, raised by 64 (1 + 128 + 128^2) to stay
            // between 0 and 2^21: base-128 digits 0 to 127
            const uint32_t x = __float_as_uint(fmaf(v[nt][8 * i + 2 * e + odd], down, 12582912.f + 1056832.f));
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              const int right = 7 * (2 - k) - 8 * e;
              w[k] |= (right >= 0 ? x >> right : x << -right) & (127u << (8 * e));
            }
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) {         // less 64, all four bytes at once: bit 6 becomes the sign
            w[k] = (w[k] ^ 0x40404040u) | ((~w[k] & 0x40404040u) << 1);
            digits[k] = __dp4a((int)w[k], 0x01010101, digits[k]);
            qf[nt][k][i][odd] = w[k];
          }
        }
      int value = (digits[0] * 128 + digits[1]) * 128 + digits[2];
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) value += __shfl_xor_sync(~0u, value, o);
      const float fh = eb == 255 ? __int_as_float(0x7fffffff) : p.scale_log2 * up + (sum - sum), fs = p.scale_log2 * sum;
      // heads 2c and 2c + 1 are lanes' g = 2c, 2c + 1
      f[nt] = two(__shfl_sync(~0u, fh, 8 * c), __shfl_sync(~0u, fh, 8 * c + 4));
      fq[nt] = two(__shfl_sync(~0u, fs, 8 * c), __shfl_sync(~0u, fs, 8 * c + 4));
#pragma unroll
      for (int e = 0; e < 2; ++e) init[nt][e] = -8 * __shfl_sync(~0u, value, 8 * c + 4 * e);
    }

    float o[NT][MT][4];
    uint64_t nM[NT], L[NT], Z[NT];              // -M, the sum of the weights and of their m', of the two heads
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      nM[nt] = two(-kFloor, -kFloor);
      L[nt] = Z[nt] = 0;
    }

    uint32_t slot = ring, fill = ring + (kStages - 1) * STAGEB;
    for (int st = first; st < t1; st += kWarps) {
      produce(st + (kStages - 1) * kWarps, fill);
      fill = slot;
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      // ---- what the 32 tokens' scales stand for, one token a lane: s, m, log2 s', 1 / s', m' / s',
      // each twice, since they are multiplied into pairs of heads
      {
        const uint32_t at = slot + OFF_SC + (lane >> 4) * 128 + (lane & 15) * 4;
        const uint32_t k0 = kva_lds32(at), v0 = kva_lds32(at + 64);
        const bool real = lane < len - st * kStep && (v0 & 0xffff) != 0;        // a scale of 0: never written, or an absent page
        const uint32_t km = real ? k0 : 0, vm = real ? v0 : 0x3c00u;
        const float2 kf = __half22float2(*reinterpret_cast<const __half2*>(&km));
        const float2 vf = __half22float2(*reinterpret_cast<const __half2*>(&vm));
        // (kf, vf: zeros, and a scale of 1 with weight 0, where there is no token)
        const float ks = kf.x, km8 = fmaf(8.f, kf.x, kf.y), ls = real ? kva_log2(vf.x) : -INFINITY;
        const float r = kva_rcp(vf.x), rz = fmaf(8.f, vf.x, vf.y) * r;
        asm volatile("st.shared.v4.f32 [%0], {%1, %1, %2, %2};" ::"r"(meta + lane * 16), "f"(ks), "f"(km8) : "memory");
        asm volatile("st.shared.v4.f32 [%0], {%1, %1, %2, %2};" ::"r"(meta + kStep * 16 + lane * 16), "f"(ls), "f"(r) : "memory");
        asm volatile("st.shared.v2.f32 [%0], {%1, %1};" ::"r"(meta + kStep * 32 + lane * 8), "f"(rz) : "memory");
      }
      __syncwarp();
      // ---- scores
      uint64_t x[2][NT][2];                     // pairs of heads of tokens tok_a and tok_a + 8 of each half
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t wa[KS], wb[KS];
        if (DP == 128) {
          const uint32_t ad = slot + h * CODEB + tok_a * ROWB + ((c * 16) ^ ((tok_a & 2) << 4));
          const uint4 a = lds128(ad), e = lds128(ad + 8 * ROWB);
          wa[0] = a.x; wa[1] = a.y; wa[KS - 2] = a.z; wa[KS - 1] = a.w;
          wb[0] = e.x; wb[1] = e.y; wb[KS - 2] = e.z; wb[KS - 1] = e.w;
        } else {
          const uint32_t ad = slot + h * CODEB + tok_a * ROWB + c * 8;
          const uint2 a = lds64(ad), e = lds64(ad + 8 * ROWB);
          wa[0] = a.x; wa[1] = a.y;
          wb[0] = e.x; wb[1] = e.y;
        }
        uint32_t a[KS][4];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          a[i][0] = wa[i] & 0x0f0f0f0fu;
          a[i][1] = wb[i] & 0x0f0f0f0fu;
          a[i][2] = (wa[i] >> 4) & 0x0f0f0f0fu;
          a[i][3] = (wb[i] >> 4) & 0x0f0f0f0fu;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // three chains side by side: one behind the other, as the starts of the next, their latency shows (249 us against 236)
          int acc[3][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {init[nt][0], init[nt][1], init[nt][0], init[nt][1]}};
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int k = 0; k < 3; ++k) kva_mma_u8s8(acc[k], a[i], qf[nt][k][i][0], qf[nt][k][i][1]);
          int sum[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[e] = (acc[0][e] * 128 + acc[1][e]) * 128 + acc[2][e];
          x[h][nt][0] = two(__int2float_rn(sum[0]), __int2float_rn(sum[1]));
          x[h][nt][1] = two(__int2float_rn(sum[2]), __int2float_rn(sum[3]));
        }
      }
      // ---- weights
      uint64_t rs[2][2], rz[2][2];
      float over = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int t = 16 * h + tok_a + 8 * r;
          uint64_t s, m, ls;
          kva_lds2(meta + t * 16, s, m);
          kva_lds2(meta + kStep * 16 + t * 16, ls, rs[h][r]);
          const uint2 z = lds64(meta + kStep * 32 + t * 8);
          rz[h][r] = two(__uint_as_float(z.x), __uint_as_float(z.y));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            x[h][nt][r] = fma2(mul2(x[h][nt][r], s), f[nt], fma2(m, fq[nt], ls));
            const float2 y = split2(add2(x[h][nt][r], nM[nt]));
            over = fmaxf(over, fmaxf(y.x, y.y));
          }
        }
      if (__any_sync(~0u, over > 8.f)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 y0 = split2(x[0][nt][0]), y1 = split2(x[0][nt][1]), y2 = split2(x[1][nt][0]), y3 = split2(x[1][nt][1]);
          const float2 old = split2(nM[nt]);
          const float M[2] = {-old.x, -old.y};
          float top[2] = {fmaxf(fmaxf(y0.x, y1.x), fmaxf(y2.x, y3.x)), fmaxf(fmaxf(y0.y, y1.y), fmaxf(y2.y, y3.y))}, k[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], s));
            top[e] = fmaxf(top[e], M[e]);
            k[e] = kva_exp2(M[e] - top[e]);
#pragma unroll
            for (int i = 0; i < MT; ++i) { o[nt][i][e] *= k[e]; o[nt][i][2 + e] *= k[e]; }
          }
          nM[nt] = two(-top[0], -top[1]);
          const uint64_t k2 = two(k[0], k[1]);
          L[nt] = mul2(L[nt], k2);
          Z[nt] = mul2(Z[nt], k2);
        }
      }
      // ---- weighted sums of the codes
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 y = split2(add2(x[h][nt][r], nM[nt]));
            const float2 w = make_float2(kva_exp2(y.x), kva_exp2(y.y));
            const uint64_t w2 = two(w.x, w.y);
            L[nt] = fma2(w2, rs[h][r], L[nt]);
            Z[nt] = fma2(w2, rz[h][r], Z[nt]);
            const __half2 h2 = __floats2half2_rn(w.x, w.y);
            pb[nt][r] = kva_transpose(*reinterpret_cast<const uint32_t*>(&h2));
          }
        const uint32_t sv = slot + (2 + h) * CODEB;
        uint32_t u[4][DP / 64];                 // tokens c, 7 - c, 8 + c, 15 - c: this lane's words
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = (j & 2) * 4 + ((j & 1) ? 7 - c : c);
          if (DP == 128) {
            const uint2 v = lds64(sv + t * ROWB + ((g * 8) ^ ((t & 2) << 4)));
            u[j][0] = v.x; u[j][DP / 64 - 1] = v.y;
          } else {
            u[j][0] = kva_lds32(sv + t * ROWB + g * 4);
          }
        }
        // row g of tile n: nibble n of one word (DP 128: word 2g, channel 16 g + n; DP 64: word g, channel 8 g + n), row g + 8:
        // of another (word 2g + 1, channel 16 g + 8 + n) or the word's upper half (channel 8 g + 4 + n)
#pragma unroll
        for (int q4 = 0; q4 < MT / 4; ++q4) {   // tiles 4 q4 .. 4 q4 + 3
          constexpr int k1 = DP / 64 - 1;
          const uint32_t sel = q4 ? 0x7632 : 0x5410, sel1 = DP == 128 ? sel : 0x7632;
          const uint32_t w[4] = {__byte_perm(u[0][0], u[1][0], sel), __byte_perm(u[0][k1], u[1][k1], sel1),
                                 __byte_perm(u[2][0], u[3][0], sel), __byte_perm(u[2][k1], u[3][k1], sel1)};
          uint32_t a[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w8 = w[k] >> 8;
            a[0][k] = kv4_pair(w[k], 0x64086408u);
            a[1][k] = kv4_pair_hi(w[k], 0xd480d480u);
            a[2][k] = kv4_pair(w8, 0x64086408u);
            a[3][k] = kv4_pair_hi(w8, 0xd480d480u);
          }
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_m16n8k16(o[nt][4 * q4 + n], a[n], pb[nt][0], pb[nt][1]);
        }
      }
      __syncwarp();                             // the slot's words are in registers of the whole warp before it is refilled
      slot = slot == ring + (kStages - 1) * STAGEB ? ring : slot + STAGEB;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- join the warps: sums over the lanes that share a head, then over the warps through shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 l2 = split2(L[nt]), z2 = split2(Z[nt]), m2 = split2(nM[nt]);
      float l[2] = {l2.x, l2.y}, z[2] = {z2.x, z2.y};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) {
          l[e] += __shfl_xor_sync(~0u, l[e], s);
          z[e] += __shfl_xor_sync(~0u, z[e], s);
        }
        if (g == 0) {
          const int h = nt * 8 + 2 * c + e;
          s_m[warp][h] = e ? -m2.y : -m2.x;
          s_l[warp][h] = l[e];
          s_z[warp][h] = z[e];
        }
      }
    }
    __syncthreads();                            // every warp has read its ring: it becomes the exchange area
    float* ex = reinterpret_cast<float*>(smem);   // [warp][head][DP]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = nt * 8 + 2 * c + (e & 1);
          const int d = DP == 128 ? 16 * g + i + ((e & 2) ? 8 : 0) : 8 * g + i + ((e & 2) ? 4 : 0);
          if (h < nh) ex[(warp * H + h) * DP + d] = o[nt][i][e];
        }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == steps;
    // parts of a list sit in the slots of their CTAs: 2 cta + 1 if the list begins in the CTA's range, else 2 cta
    const int my_slot = 2 * (int)blockIdx.x + (t0 == 0 ? 1 : 0);
    for (int i = tid; i < nh * DP; i += kThreads) {
      const int h = i / DP, d = i - h * DP;
      float top = s_m[0][h];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][h]);
      float acc = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float k = kva_exp2(s_m[w][h] - top);
        acc = fmaf(k, ex[(w * H + h) * DP + d] + s_z[w][h], acc);
        l = fmaf(k, s_l[w][h], l);
      }
      if (whole) {
        if (d < p.dv) kva_store(p.out, ((int64_t)b * p.heads + head0 + h) * p.dv + d, p.bf16, l == 0.f ? 0.f : acc / l);
      } else {
        float* dst = p.part + ((size_t)my_slot * H + h) * PSTR;
        dst[d] = acc;
        if (d == 0) { dst[DP] = top; dst[DP + 1] = l; }
      }
    }
    if (!whole) {
      // CTAs of this list: the ones whose ranges hold its first and its last step
      const int c0 = (int)(((list_begin + (unit ? 0 : kOpen) + 1) * ctas - 1) / N), c1 = (int)(((list_begin + size) * ctas - 1) / N);
      __syncthreads();
      if (tid == 0) {                           // behind the barrier its fence speaks for the whole CTA
        __threadfence();
        s_last = atomicAdd(p.tickets + c0, 1) == c1 - c0;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        kva_join_parts<DP, H>(p, (int64_t)b * p.heads + head0, nh, c0, c1);
        if (tid == 0) p.tickets[c0] = 0;
      }
    }
    __syncthreads();                            // the exchange area becomes the ring again
  }
  if (bad_page && p.status_word) atomicOr(p.status_word, UNIQL_STATUS_BAD_INDEX);
}

template <int DP, int NT>
static constexpr size_t kva_smem() {
  const size_t ring = (size_t)kva::kWarps * (kva::kStages * (32 * DP + 256) + kva::kStep * 40);
  const size_t ex = (size_t)kva::kWarps * 8 * NT * DP * 4;
  return ring > ex ? ring : ex;
}

static int kva_ctas(int nt) {
  const int n = device_info().sm_count * kva::per_sm(nt);
  return n < kva::kMaxCtas ? n : kva::kMaxCtas;
}
static int kva_nt(int64_t heads, int64_t kv_heads) { return heads / kv_heads > 8 ? 2 : 1; }

template <int DP, int NT, bool PAGE16>
static int kva_launch(KvaParams& p, cudaStream_t stream) {
  static thread_local bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    UNIQL_CUDA_TRY(cudaFuncSetAttribute(kv4_attention_kernel<DP, NT, PAGE16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)kva_smem<DP, NT>()));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return launch_pdl(kv4_attention_kernel<DP, NT, PAGE16>, (unsigned)kva_ctas(NT), kva::kThreads, kva_smem<DP, NT>(), stream, p);
}

}  // namespace uniql

extern "C" size_t uniql_kv4_attention_scratch_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dp) {
  using namespace uniql;
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || (dp != 64 && dp != 128)) return 0;
  const int nt = kva_nt(heads, kv_heads);
  return UNIQL_SCRATCH_COUNTER_BYTES + (size_t)2 * kva_ctas(nt) * 8 * nt * (dp + 4) * sizeof(float);
}

extern "C" int uniql_kv4_attention(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* codes,
                                   const void* scales, int64_t num_pages, int64_t page_size, int64_t dp,
                                   const int32_t* block_table, int64_t ld_table, int64_t max_blocks, const int32_t* lens,
                                   int64_t batch, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, float softmax_scale,
                                   int dtype, void* out, void* scratch, size_t scratch_bytes, int* status_word, void* stream) {
  using namespace uniql;
  static_assert(kva::kMaxCtas * sizeof(int) <= UNIQL_SCRATCH_COUNTER_BYTES, "a ticket per CTA");
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || num_pages < 0 || dk <= 0 || dv <= 0 || max_blocks < 0 || ld_table < max_blocks)
    return UNIQL_EINVAL;
  if (dtype != UNIQL_F16 && dtype != UNIQL_BF16) return UNIQL_EDTYPE;
  int st = kv4_check(num_pages, page_size, dp, kv_heads, dk, dv);
  if (st != UNIQL_OK) return st;
  if (heads % kv_heads || heads > 16384 || batch > UNIQL_KV_MAX_BATCH || max_blocks > kMaxTokens) return UNIQL_ESHAPE;
  if (!(softmax_scale > 0.f) || softmax_scale > 1e30f) return UNIQL_EINVAL;
  if (batch == 0) return UNIQL_OK;
  if (!q || !lens || !out || (max_blocks > 0 && !block_table)) return UNIQL_EINVAL;
  if (num_pages > 0 && (!codes || !scales || !aligned16(codes) || !aligned16(scales))) return UNIQL_EINVAL;
  if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255u) ||
      scratch_bytes < uniql_kv4_attention_scratch_bytes(batch, heads, kv_heads, dp))
    return UNIQL_ESCRATCH;
  KvaParams p;
  p.q = (const unsigned char*)q; p.q_bs = q_batch_stride; p.q_hs = q_head_stride;
  // without pages every copy is of no bytes, but from an address that exists
  p.codes = (const unsigned char*)(num_pages ? codes : scratch); p.scales = (const unsigned char*)(num_pages ? scales : scratch);
  p.table = block_table; p.ld_table = ld_table; p.lens = lens; p.out = (unsigned char*)out;
  p.tickets = (int*)scratch; p.part = (float*)((char*)scratch + UNIQL_SCRATCH_COUNTER_BYTES); p.status_word = status_word;
  const int nt = kva_nt(heads, kv_heads);
  p.batch = (int)batch; p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.group = (int)(heads / kv_heads);
  p.hgroups = (p.group + 8 * nt - 1) / (8 * nt);
  p.max_blocks = (int)max_blocks; p.num_pages = (int)num_pages; p.page_shift = page_shift_of(page_size);
  p.dk = (int)dk; p.dv = (int)dv; p.bf16 = dtype == UNIQL_BF16;
  p.q_vec = aligned16(q) && !((q_batch_stride | q_head_stride) & 7);
  p.scale_log2 = softmax_scale * 1.44269504088896340736f;
  cudaStream_t s = (cudaStream_t)stream;
  auto launch = [&](auto small) {
    constexpr bool P16 = decltype(small)::value;
    if (dp == 128) return nt == 1 ? kva_launch<128, 1, P16>(p, s) : kva_launch<128, 2, P16>(p, s);
    return nt == 1 ? kva_launch<64, 1, P16>(p, s) : kva_launch<64, 2, P16>(p, s);
  };
  return page_size == 16 ? launch(std::true_type{}) : launch(std::false_type{});
}
