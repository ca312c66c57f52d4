// The paged 4-bit KV cache: planning of its pages, the quantising write and the dequantising read.  Layout and rules:
// include/uniql_b200.h.  No counterpart in UniQL.
#include "common.cuh"
#include "kv_cache.cuh"

namespace uniql {

// ------------------------------------------------------------------------------------------------ page plan
// need_i = ceil((len_i + new_i) / P) - ceil(len_i / P), cut at the width of the table; the exclusive sums of need and new
// say which entries of the free stack and which places of the packed tokens a request owns.  Every CTA computes both sums
// for the whole batch (8 bytes a request from L2) and keeps them in shared memory; the new pages and the new tokens are then
// flat lists that all threads walk, each finding its request by bisection, so that one prompt of thousands of tokens costs no
// more than thousands of single ones.  lens and free_count may be overwritten in place, so what goes there waits for every CTA's
// reads: up to 8 CTAs are one cluster with a barrier; a step of more tokens than those have threads for takes a grid over the
// GPU and a second launch of one CTA (257328 tokens of 1024 requests: 35 us in one cluster, 9.5 as grid and second launch).
//
// A step's plan (cu_keys given) serves whole requests: one that cannot have all its pages, columns and places keeps its length and
// takes nothing.  What is impossible by itself does not count for the others; of the rest, the ones whose inclusive sums stay within
// the stack and the places are served.  A later request that needs a page sums to more than an earlier one that was left out, so the
// served ones' pages are the first of the list and s_first holds for them as it is.  s_len of a request left out is ~len.
constexpr int kPlanThreads = 1024, kPlanCap = 1 << 30;

struct PlanParams {
  const int32_t* lens;
  const int32_t* new_lens;
  int32_t* table;
  int64_t ld_table;
  const int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int64_t* positions;
  int32_t* cu_new;
  int32_t* lens_out;
  int32_t* free_count_out;
  int* status_word;
  int32_t* key_lens;                            // of a step's plan: keys of each request, and their exclusive sums
  int32_t* cu_keys;
  int64_t total_new;
  int batch, max_blocks, free_cap, page_shift;
  int lists, totals;                            // what this launch does: pages and tokens; lengths, starts and count
};

// largest i with start[i] <= x, for start[0] = 0 <= x
__device__ __forceinline__ int plan_find(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv_page_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int plan_smem[];
  int* s_len = plan_smem;                       // [batch]
  int* s_cu = s_len + p.batch;                  // [batch + 1]
  int* s_first = s_cu + p.batch + 1;            // [batch + 1]
  __shared__ long long warp_new[32], warp_need[32];
  __shared__ long long carry_new, carry_need, carry_keys;
  __shared__ int s_count, s_taken;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pmask = (1 << p.page_shift) - 1;
  if (tid == 0) {
    carry_new = carry_need = carry_keys = 0;
    s_taken = 0;
    s_cu[0] = s_first[0] = 0;                   // all there is of them when the batch is empty
    s_count = min(max(p.free_count[0], 0), p.free_cap);
  }
  const bool whole = p.cu_keys != nullptr, sums = whole && p.totals && blockIdx.x == 0;
  bool short_table = false;
  __syncthreads();
  for (int i0 = 0; i0 < p.batch; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int len = 0, add = 0, need = 0;
    bool out = false;                           // not served by a step's plan
    if (i < p.batch) {
      len = min(max(p.lens[i], 0), kMaxTokens);
      add = min(max(p.new_lens[i], 0), kMaxTokens);
      const int had = (len + pmask) >> p.page_shift, has = (len + add + pmask) >> p.page_shift;
      need = max(min(has, p.max_blocks) - had, 0);
      if (whole) {
        out = (has > p.max_blocks && add > 0) || need > s_count;
        if (out) need = 0;
      } else {
        short_table |= has > p.max_blocks && add > 0;
        s_len[i] = len;
      }
    }
    long long xn = add, xb = need;              // inclusive sums over the warp, then over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(~0u, xn, o), b = __shfl_up_sync(~0u, xb, o);
      if (lane >= o) { xn += a; xb += b; }
    }
    if (lane == 31) { warp_new[warp] = xn; warp_need[warp] = xb; }
    __syncthreads();
    if (warp == 0) {
      long long a = warp_new[lane], b = warp_need[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long c = __shfl_up_sync(~0u, a, o), d = __shfl_up_sync(~0u, b, o);
        if (lane >= o) { a += c; b += d; }
      }
      warp_new[lane] = a;
      warp_need[lane] = b;
    }
    __syncthreads();
    const long long bn = carry_new + (warp ? warp_new[warp - 1] : 0), bb = carry_need + (warp ? warp_need[warp - 1] : 0);
    // sums of lengths that nobody can mean stop at kPlanCap: the lists below stay sorted, and places under it are exact
    if (i < p.batch) {
      s_cu[i] = (int)min(bn + xn - add, (long long)kPlanCap);
      s_first[i] = (int)min(bb + xb - need, (long long)kPlanCap);
    }
    if (whole && i < p.batch) {
      out |= (add > 0 && bn + xn > p.total_new) || (need > 0 && bb + xb > s_count);
      if (!out && need > 0) atomicMax(&s_taken, (int)(bb + xb));
      short_table |= out;
      s_len[i] = out ? ~len : len;
    }
    __syncthreads();
    if (sums) {
      const int keys = i < p.batch && !out ? len + add : 0;
      long long xk = keys;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(~0u, xk, o);
        if (lane >= o) xk += v;
      }
      // bn and bb of this round have been taken: the warps' sums may go
      if (lane == 31) warp_need[warp] = xk;
      __syncthreads();
      long long bk = lane < warp ? warp_need[lane] : 0;
#pragma unroll
      for (int o = 16; o; o >>= 1) bk += __shfl_xor_sync(~0u, bk, o);
      bk += carry_keys;
      if (i < p.batch) {
        p.key_lens[i] = keys;
        p.cu_keys[i] = (int)min(bk + xk - keys, (long long)kPlanCap);
        if (i == p.batch - 1) p.cu_keys[p.batch] = (int)min(bk + xk, (long long)kPlanCap);
      }
      __syncthreads();
      if (tid == kPlanThreads - 1) carry_keys = bk + xk;
    }
    if (tid == kPlanThreads - 1) {
      carry_new = bn + xn;
      carry_need = bb + xb;
      s_cu[min(i0 + kPlanThreads, p.batch)] = (int)min(carry_new, (long long)kPlanCap);      // the next round writes the same value
      s_first[min(i0 + kPlanThreads, p.batch)] = (int)min(carry_need, (long long)kPlanCap);
    }
    __syncthreads();
  }
  if (sums && p.batch == 0 && tid == 0) p.cu_keys[0] = 0;
  const int tokens = s_cu[p.batch], count = s_count, pages = whole ? s_taken : s_first[p.batch];
  const int rank = blockIdx.x, ranks = gridDim.x, step = ranks * kPlanThreads;
  if (p.lists) {
  for (int x = rank * kPlanThreads + tid; x < pages; x += step) {
    const int i = plan_find(s_first, p.batch, x);       // a served one: theirs are the first places
    const int had = (s_len[i] + pmask) >> p.page_shift;
    p.table[(size_t)i * p.ld_table + had + (x - s_first[i])] = x < count ? p.free_pages[count - 1 - x] : -1;
  }
  for (int64_t x = (int64_t)rank * kPlanThreads + tid; x < p.total_new; x += step) {
    int64_t slot = -1, pos = 0;
    if (x < tokens) {
      const int i = plan_find(s_cu, p.batch, (int)x);
      const int held = s_len[i], len = held < 0 ? ~held : held, at = len + ((int)x - s_cu[i]);
      const int had = (len + pmask) >> p.page_shift, block = at >> p.page_shift;
      int page = -1;
      if (held >= 0 && block < p.max_blocks) {
        const int r = s_first[i] + block - had;
        if (block < had) page = p.table[(size_t)i * p.ld_table + block];
        else if (r < count) page = p.free_pages[count - 1 - r];
      }
      pos = at;
      if (page >= 0) slot = ((int64_t)page << p.page_shift) + (at & pmask);
    }
    p.slots[x] = slot;
    p.positions[x] = pos;
  }
  if ((short_table || (rank == 0 && tid == 0 && (pages > count || tokens > p.total_new))) && p.status_word)
    atomicOr(p.status_word, UNIQL_STATUS_NO_PAGE);
  }
  if (!p.totals) return;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0) {
    for (int i = tid; i <= p.batch; i += kPlanThreads) {
      p.cu_new[i] = whole ? (int)min((int64_t)s_cu[i], p.total_new) : s_cu[i];
      if (i < p.batch) p.lens_out[i] = s_len[i] < 0 ? ~s_len[i] : s_len[i] + min(max(p.new_lens[i], 0), kMaxTokens);
    }
    if (tid == 0) p.free_count_out[0] = max(count - pages, 0);
  }
}

// ------------------------------------------------------------------------------------------------ append
// A row (one token, one head) is DP / 16 lanes with sixteen channels each: two 16-byte loads, the extremes over the lanes
// (least value and negated greatest one as a 16-bit pair: one shuffle a level), two packed words stored.  HBM-bound by the
// reads, 4 bytes a channel against 0.5 written, if the instructions are few: the packed minimum carries NaN along, the codes
// are rounded by adding 1.5 * 2^23 and joined as the low bits of those sums, and sixteen channels a lane share what a row costs
// (eight: 50 us for 14760 tokens of 8 heads, 60 MB read; sixteen: 34; with K's and V's rows in one turn and packed
// arithmetic: 27; exact comparisons for the channels near a half-way point alone, not for their whole word: 24).
// (hi - lo) / 15 is the quotient by the reciprocal and one
// residual step (Markstein), equal to the division for every mantissa.
//
// Codes are taken from a quotient in fp32.  Where that leaves the side of a half-way point open, the two sides are compared
// exactly: x - z spans at most 41 bits and (k + 1/2) * s sixteen, both exact in fp64.
constexpr float kRound = 12582912.f;            // 1.5 * 2^23
__device__ __noinline__ uint32_t kv4_exact_code(float x, float z, float s, float y) {
  // y: the quotient within 2^-22 (relative), so its integer part lies on the right side of the half-way point below it
  const float k = floorf(fminf(fmaxf(y, 0.f), 15.f));
  const double d = (double)x - (double)z, mid = ((double)k + 0.5) * (double)s;
  const int ki = (int)k;
  return (uint32_t)min(d > mid || (d == mid && (ki & 1)) ? ki + 1 : ki, 15);
}

struct AppendParams {
  const unsigned char* src[2];
  int64_t token_stride[2], head_stride[2];      // elements
  const int64_t* slots;
  uint32_t* codes;
  __half2* scales;
  int* status_word;
  int64_t num_slots;
  uint32_t rows;                                // tokens * heads, below 2^31
  FastDiv heads;
  int d[2], page_shift;
};

constexpr int kAppendThreads = 256, kAppendCtas = 6;      // CTAs an SM holds

template <bool BF16>
struct Pair16 {
  using T = __half2;
};
template <>
struct Pair16<true> {
  using T = __nv_bfloat162;
};

template <int DP, bool BF16>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int W = DP / 16;                    // lanes of a row
  using T2 = typename Pair16<BF16>::T;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t sub = threadIdx.x % W;
  const uint32_t step = gridDim.x * (kAppendThreads / W);
  const uint32_t kInfs = BF16 ? 0x7f807f80u : 0x7c007c00u;
  // the lanes of a warp stay in the loop together: the shuffles below name the whole warp
  const uint32_t first = blockIdx.x * (kAppendThreads / W) + threadIdx.x / W, ahead = (threadIdx.x % 32) / W;
  for (uint32_t r = first; r - ahead < p.rows; r += step) {
    const bool live = r < p.rows;
    const uint32_t t = live ? p.heads.quot(r) : 0, h = live ? r - t * p.heads.d : 0;
    const int64_t slot = live ? p.slots[t] : -1;
    const bool stored = slot >= 0 && slot < p.num_slots;
    if (live && !stored && slot != -1 && sub == 0 && p.status_word) atomicOr(p.status_word, UNIQL_STATUS_BAD_INDEX);
    // K's row and V's row of the token and head: one index, both loads in flight
    uint4 raws[2][2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const unsigned char* src = p.src[kv] + 2 * (t * p.token_stride[kv] + h * p.head_stride[kv] + sub * 16);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        raws[kv][j] = make_uint4(0, 0, 0, 0);
        if (stored && (int)sub * 16 + 8 * j < p.d[kv]) raws[kv][j] = *reinterpret_cast<const uint4*>(src + 16 * j);
      }
    }
    const int64_t krow = ((((slot >> p.page_shift) * 2) * p.heads.d + h) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
    const uint4 (&raw)[2] = raws[kv];
    const bool mine[2] = {stored && (int)sub * 16 < p.d[kv], stored && (int)sub * 16 + 8 < p.d[kv]};
    // (least, -greatest) of the row; places without channels hold infinities
    uint32_t eb = kInfs;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      T2 least = *reinterpret_cast<const T2*>(&u[0]), most = least;
#pragma unroll
      for (int e = 1; e < 4; ++e) {
        least = __hmin2_nan(least, *reinterpret_cast<const T2*>(&u[e]));
        most = __hmax2_nan(most, *reinterpret_cast<const T2*>(&u[e]));
      }
      T2 ends;
      ends.x = __hmin_nan(least.x, least.y);
      ends.y = __hneg(__hmax_nan(most.x, most.y));
      if (mine[j]) {
        ends = __hmin2_nan(ends, *reinterpret_cast<const T2*>(&eb));
        eb = *reinterpret_cast<const uint32_t*>(&ends);
      }
    }
#pragma unroll
    for (int o = W / 2; o; o >>= 1) {
      const uint32_t other = __shfl_xor_sync(~0u, eb, o);
      const T2 ends = __hmin2_nan(*reinterpret_cast<const T2*>(&eb), *reinterpret_cast<const T2*>(&other));
      eb = *reinterpret_cast<const uint32_t*>(&ends);
    }
    const T2 ends = *reinterpret_cast<const T2*>(&eb);
    float lo, hi;
    if constexpr (BF16) {
      lo = __bfloat162float(ends.x);
      hi = -__bfloat162float(ends.y);
    } else {
      lo = __half2float(ends.x);
      hi = -__half2float(ends.y);
    }
    const bool nan = lo != lo || hi != hi, wide = lo < -65504.f || hi > 65504.f;
    lo = fminf(fmaxf(lo, -65504.f), 65504.f);
    hi = fminf(fmaxf(hi, -65504.f), 65504.f);
    constexpr float k15 = 1.f / 15.f;
    const float span = hi - lo, q0 = span * k15;
    __half sh = __float2half_rn(fmaf(fmaf(-15.f, q0, span), k15, q0));
    if (__half2float(sh) < 5.9604645e-8f) sh = __ushort_as_half(1);      // 2^-24: a scale is never zero
    __half zh = __float2half_rn(lo);
    const float s = __half2float(sh), z = __half2float(zh);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    // The usual row: y = x / s - z / s in one fused step, which is within 2^-17 of the quotient while |z / s| is at most 64, and no
    // quotient leaves 0..15 by half a step (z is the minimum itself, s is off by less than 1/30).  Any other row takes the exact
    // comparisons throughout, as does a half row with a quotient near a half-way point.
    const float zi = -z * inv;
    const bool odd = wide || z != lo || fabsf(zi) > 64.f || s < 1e-6f;
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (!mine[j] || nan) continue;
      const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      float far = odd ? 1.f : 0.f;
      constexpr uint32_t kBits = 0x4b400000u;   // of kRound; what eight of them add to the word:
      constexpr uint32_t kAll = kBits + (kBits << 4) + (kBits << 8) + (kBits << 12) + (kBits << 16) + (kBits << 20) + (kBits << 24) + (kBits << 28);
      uint32_t w = 0u - kAll;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 f;
        if constexpr (BF16) f = __bfloat1622float2(*reinterpret_cast<const T2*>(&u[e]));
        else f = __half22float2(*reinterpret_cast<const T2*>(&u[e]));
        const uint64_t y = fma2(two(f.x, f.y), two(inv, inv), two(zi, zi)), up = add2(y, two(kRound, kRound));
        const float2 off = split2(fma2(add2(up, two(-kRound, -kRound)), two(-1.f, -1.f), y)), n = split2(up);
        far = fmaxf(far, fmaxf(fabsf(off.x), fabsf(off.y)));
        w += (__float_as_uint(n.x) << (8 * e)) + (__float_as_uint(n.y) << (8 * e + 4));
      }
      if (far > 0.49998f) {                     // some quotient within 2e-5 of a half-way point, or an odd row
        w = 0;
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const uint32_t ue = (e >> 1) == 0 ? u[0] : (e >> 1) == 1 ? u[1] : (e >> 1) == 2 ? u[2] : u[3];
          float xe = BF16 ? __uint_as_float((e & 1) ? ue & 0xffff0000u : ue << 16)
                          : __half2float(__ushort_as_half((unsigned short)(ue >> (16 * (e & 1)))));
          const float y = fmaf(xe, inv, zi), n = rintf(y);
          if (!odd && fabsf(y - n) <= 0.49998f) {
            w |= (uint32_t)(int)n << (4 * e);
            continue;
          }
          xe = fminf(fmaxf(xe, -65504.f), 65504.f);
          w |= kv4_exact_code(xe, z, s, (xe - z) * inv) << (4 * e);
        }
      }
      word[j] = w;
    }
    if (stored) {
      const int64_t row = krow + (kv ? (int64_t)p.heads.d << p.page_shift : 0);
      *reinterpret_cast<uint2*>(p.codes + row * (DP / 8) + 2 * sub) = make_uint2(word[0], word[1]);
      if (sub == 0) {
        if (nan) sh = zh = __ushort_as_half(0x7fff);
        p.scales[row] = __halves2half2(sh, zh);
      }
    }
    }
  }
}

// ------------------------------------------------------------------------------------------------ gather
// zero + scale * code, fused so that it is rounded once, from the packed rows of a token range.  HBM-bound by the writes.
// A CTA owns 4, 8 or 16 packed places: one thread per place finds request, page and row (bisection over cu, the batch's last
// narrowing in shared memory), then all walk the places' rows, DP / 8 lanes a row, one word in and 16 bytes out each.
constexpr int kGatherThreads = 256, kGatherTokens = 16, kGatherRows = 4, kGatherCu = 1024;

struct GatherParams {
  const uint32_t* codes;
  const __half2* scales;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* cu;
  unsigned char* out[2];
  int* status_word;
  int64_t ld_table, num_pages, total;
  FastDiv heads;
  int batch, max_blocks, d[2], page_shift;
  int tokens;                                   // places of a CTA, at most kGatherTokens
};

template <int DP, bool BF16>
__global__ void __launch_bounds__(kGatherThreads) kv4_gather_kernel(const __grid_constant__ GatherParams p) {
  constexpr int W = DP / 8, ROWS = kGatherThreads / W;
  __shared__ int64_t s_row[kGatherTokens];      // row of head 0 of K on the token's page, or -1
  __shared__ int s_cu[kGatherCu + 1];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int heads = p.heads.d;
  const bool local = p.batch <= kGatherCu;
  if (local)
    for (int i = threadIdx.x; i <= p.batch; i += kGatherThreads) s_cu[i] = p.cu[i];
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.batch > 0 && p.status_word) {
    const int32_t* cu = local ? s_cu : p.cu;
    if (cu[0] < 0 || cu[p.batch] > p.total) atomicOr(p.status_word, UNIQL_STATUS_BAD_INDEX);       // tokens that have no place
  }
  if (threadIdx.x < p.tokens) {
    const int32_t* cu = local ? s_cu : p.cu;
    const int64_t t = t0 + threadIdx.x;
    int64_t row = -1;
    if (t < p.total && p.batch > 0 && t >= cu[0] && t < cu[p.batch]) {
      int lo = 0, hi = p.batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int64_t at = t - cu[lo] + (p.starts ? max(p.starts[lo], 0) : 0);
      const int64_t block = at >> p.page_shift;
      int page = -1;
      if (block < p.max_blocks) page = p.table[(size_t)lo * p.ld_table + block];
      if (page >= 0 && page < p.num_pages) row = (((int64_t)page * 2 * heads) << p.page_shift) + (at & ((1 << p.page_shift) - 1));
      else if (p.status_word) atomicOr(p.status_word, UNIQL_STATUS_BAD_INDEX);
    }
    s_row[threadIdx.x] = row;
  }
  __syncthreads();
  const uint32_t n = (uint32_t)(p.total - t0 < p.tokens ? p.total - t0 : p.tokens);
  const uint32_t sub = threadIdx.x % W;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint32_t d = p.d[kv];
    if (sub * 8 >= d) continue;
    unsigned char* out = p.out[kv] + 2 * (t0 * heads * d + sub * 8);
    const uint32_t* codes = p.codes + sub;
    const int64_t shift_rows = kv ? (int64_t)heads << p.page_shift : 0;
    for (uint32_t r0 = threadIdx.x / W; r0 < n * heads; r0 += kGatherRows * ROWS) {
      uint32_t w[kGatherRows];
      __half2 sz[kGatherRows];
#pragma unroll
      for (int j = 0; j < kGatherRows; ++j) {
        const uint32_t r = r0 + j * ROWS;
        w[j] = 0;
        sz[j] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
        if (r < n * heads) {
          const uint32_t i = p.heads.quot(r), h = r - i * heads;
          if (s_row[i] >= 0) {
            const int64_t row = s_row[i] + shift_rows + ((int64_t)h << p.page_shift);
            w[j] = codes[row * W];
            sz[j] = p.scales[row];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kGatherRows; ++j) {
        const uint32_t r = r0 + j * ROWS;
        if (r >= n * heads) break;
        uint4 o;
        uint32_t c[4];
        kv4_codes(w[j], c);                     // (d, d + 4) pairs; absent rows are 0 + 0 * 0
        if constexpr (!BF16) {
          const __half2 s2 = __low2half2(sz[j]), z2 = __high2half2(sz[j]);
          uint32_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 f = __hfma2(*reinterpret_cast<const __half2*>(&c[e]), s2, z2);
            v[e] = *reinterpret_cast<const uint32_t*>(&f);
          }
          o = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                         __byte_perm(v[2], v[3], 0x7632));
        } else {
          const float s = __low2float(sz[j]), z = __high2float(sz[j]);
          float v[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&c[e]));
            v[e] = fmaf(f.x, s, z);
            v[e + 4] = fmaf(f.y, s, z);
          }
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
            u[e] = *reinterpret_cast<const uint32_t*>(&b);
          }
          o = make_uint4(u[0], u[1], u[2], u[3]);
        }
        *reinterpret_cast<uint4*>(out + (size_t)(2 * r) * d) = o;
      }
    }
  }
}

}  // namespace uniql

// ------------------------------------------------------------------------------------------------ C ABI
static int kv_plan(const int32_t* lens, const int32_t* new_lens, int64_t batch, int32_t* block_table, int64_t ld_table,
                   int64_t max_blocks, const int32_t* free_pages, int64_t free_cap, const int32_t* free_count, int64_t page_size,
                   int64_t total_new, int64_t* slots, int64_t* positions, int32_t* cu_new, int32_t* lens_out,
                   int32_t* free_count_out, int32_t* key_lens, int32_t* cu_keys, int* status_word, void* stream) {
  using namespace uniql;
  if (batch < 0 || total_new < 0 || max_blocks < 0 || free_cap < 0 || ld_table < max_blocks) return UNIQL_EINVAL;
  const int shift = page_shift_of(page_size);
  if (shift < 0 || batch > UNIQL_KV_MAX_BATCH || total_new > kMaxTokens || max_blocks > kMaxTokens || free_cap > kMaxTokens)
    return UNIQL_ESHAPE;
  if (!cu_new || !free_count || !free_count_out) return UNIQL_EINVAL;
  if (batch > 0 && (!lens || !new_lens || !lens_out || (max_blocks > 0 && !block_table))) return UNIQL_EINVAL;
  if ((total_new > 0 && (!slots || !positions)) || (free_cap > 0 && !free_pages)) return UNIQL_EINVAL;
  PlanParams p;
  p.lens = lens; p.new_lens = new_lens; p.table = block_table; p.ld_table = ld_table;
  p.free_pages = free_pages; p.free_count = free_count; p.slots = slots; p.positions = positions;
  p.cu_new = cu_new; p.lens_out = lens_out; p.free_count_out = free_count_out; p.status_word = status_word;
  p.key_lens = key_lens; p.cu_keys = cu_keys;
  p.total_new = total_new; p.batch = (int)batch; p.max_blocks = (int)max_blocks; p.free_cap = (int)free_cap; p.page_shift = shift;
  const size_t smem = (3 * (size_t)batch + 2) * sizeof(int);
  // raised for every size: what a kernel gets by default counts its static shared memory too
  static thread_local bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    UNIQL_CUDA_TRY(cudaFuncSetAttribute(kv_page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (3 * UNIQL_KV_MAX_BATCH + 2) * (int)sizeof(int)));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t ctas = (total_new + kPlanThreads - 1) / kPlanThreads;
  auto launch = [&](int64_t grid, int cluster, int lists, int totals) {
    p.lists = lists;
    p.totals = totals;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;         // a cluster launch costs the host 3 us more
    UNIQL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_page_plan_kernel, (const PlanParams&)p));
    return (int)UNIQL_OK;
  };
  if (ctas <= 8) return launch(ctas < 1 ? 1 : ctas, ctas < 1 ? 1 : (int)ctas, 1, 1);
  const int64_t sms = device_info().sm_count;
  const int st = launch(ctas < sms ? ctas : sms, 1, 1, 0);
  return st != UNIQL_OK ? st : launch(1, 1, 0, 1);
}

extern "C" int uniql_kv_page_plan(const int32_t* lens, const int32_t* new_lens, int64_t batch, int32_t* block_table,
                                  int64_t ld_table, int64_t max_blocks, const int32_t* free_pages, int64_t free_cap,
                                  const int32_t* free_count, int64_t page_size, int64_t total_new, int64_t* slots,
                                  int64_t* positions, int32_t* cu_new, int32_t* lens_out, int32_t* free_count_out,
                                  int* status_word, void* stream) {
  return kv_plan(lens, new_lens, batch, block_table, ld_table, max_blocks, free_pages, free_cap, free_count, page_size, total_new,
                 slots, positions, cu_new, lens_out, free_count_out, nullptr, nullptr, status_word, stream);
}

extern "C" int uniql_kv_step_plan(const int32_t* lens, const int32_t* new_lens, int64_t batch, int32_t* block_table,
                                  int64_t ld_table, int64_t max_blocks, const int32_t* free_pages, int64_t free_cap,
                                  const int32_t* free_count, int64_t page_size, int64_t total_new, int64_t* slots,
                                  int64_t* positions, int32_t* cu_new, int32_t* lens_out, int32_t* free_count_out,
                                  int32_t* key_lens, int32_t* cu_keys, int* status_word, void* stream) {
  if (!cu_keys || (batch > 0 && !key_lens)) return UNIQL_EINVAL;
  return kv_plan(lens, new_lens, batch, block_table, ld_table, max_blocks, free_pages, free_cap, free_count, page_size, total_new,
                 slots, positions, cu_new, lens_out, free_count_out, key_lens, cu_keys, status_word, stream);
}

extern "C" int uniql_kv4_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t tokens, int64_t kv_heads,
                                int64_t dk, int64_t dv, const int64_t* slots, void* codes, void* scales, int64_t num_pages,
                                int64_t page_size, int64_t dp, int* status_word, void* stream) {
  using namespace uniql;
  if (tokens < 0 || kv_heads <= 0 || num_pages < 0 || dk <= 0 || dv <= 0) return UNIQL_EINVAL;
  if (dtype != UNIQL_F16 && dtype != UNIQL_BF16) return UNIQL_EDTYPE;
  const int st = kv4_check(num_pages, page_size, dp, kv_heads, dk, dv);
  if (st != UNIQL_OK) return st;
  if (tokens > kMaxTokens) return UNIQL_ESHAPE;
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return UNIQL_EINVAL;
  if (tokens == 0) return UNIQL_OK;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v)) return UNIQL_EINVAL;
  if (num_pages > 0 && (!codes || !scales || !aligned16(codes) || !aligned16(scales))) return UNIQL_EINVAL;
  AppendParams p;
  p.token_stride[0] = k_token_stride; p.token_stride[1] = v_token_stride;
  p.head_stride[0] = k_head_stride; p.head_stride[1] = v_head_stride;
  p.codes = (uint32_t*)codes; p.scales = (__half2*)scales; p.status_word = status_word;
  p.num_slots = num_pages * page_size; p.heads = FastDiv((uint32_t)kv_heads); p.d[0] = (int)dk; p.d[1] = (int)dv;
  p.page_shift = page_shift_of(page_size);
  const bool bf16 = dtype == UNIQL_BF16;
  auto kernel = dp == 128 ? (bf16 ? kv4_append_kernel<128, true> : kv4_append_kernel<128, false>)
                          : (bf16 ? kv4_append_kernel<64, true> : kv4_append_kernel<64, false>);
  const int64_t per = kAppendThreads / (dp / 16), cap = 4 * kAppendCtas * (int64_t)device_info().sm_count;     // four waves even out: 27 us against 30 of one
  const int64_t slab = ((int64_t)1 << 30) / kv_heads;                   // tokens of a launch: rows stay below 2^31
  for (int64_t t0 = 0; t0 < tokens; t0 += slab) {
    const int64_t n = tokens - t0 < slab ? tokens - t0 : slab;
    p.src[0] = (const unsigned char*)k + 2 * t0 * k_token_stride;
    p.src[1] = (const unsigned char*)v + 2 * t0 * v_token_stride;
    p.slots = slots + t0;
    p.rows = (uint32_t)(n * kv_heads);
    const int64_t ctas = ((int64_t)p.rows + per - 1) / per;
    const int err = launch_pdl(kernel, (unsigned)(ctas < cap ? ctas : cap), kAppendThreads, 0, (cudaStream_t)stream, p);
    if (err != UNIQL_OK) return err;
  }
  return UNIQL_OK;
}

extern "C" int uniql_kv4_gather(const void* codes, const void* scales, int64_t num_pages, int64_t page_size, int64_t dp,
                                int64_t kv_heads, const int32_t* block_table, int64_t ld_table, int64_t max_blocks,
                                int64_t batch, const int32_t* starts, const int32_t* cu, int64_t total, int64_t dk, int64_t dv,
                                int dtype, void* k_out, void* v_out, int* status_word, void* stream) {
  using namespace uniql;
  if (total < 0 || batch < 0 || kv_heads <= 0 || num_pages < 0 || dk <= 0 || dv <= 0 || max_blocks < 0 || ld_table < max_blocks)
    return UNIQL_EINVAL;
  if (dtype != UNIQL_F16 && dtype != UNIQL_BF16) return UNIQL_EDTYPE;
  const int st = kv4_check(num_pages, page_size, dp, kv_heads, dk, dv);
  if (st != UNIQL_OK) return st;
  if (total > kMaxTokens || batch > kMaxTokens || max_blocks > kMaxTokens) return UNIQL_ESHAPE;
  if (total == 0) return UNIQL_OK;
  if (!k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) return UNIQL_EINVAL;
  if (batch > 0 && (!cu || (max_blocks > 0 && !block_table))) return UNIQL_EINVAL;
  if (num_pages > 0 && (!codes || !scales || !aligned16(codes) || !aligned16(scales))) return UNIQL_EINVAL;
  GatherParams p;
  p.codes = (const uint32_t*)codes; p.scales = (const __half2*)scales; p.table = block_table; p.starts = starts; p.cu = cu;
  p.out[0] = (unsigned char*)k_out; p.out[1] = (unsigned char*)v_out; p.status_word = status_word;
  p.ld_table = ld_table; p.num_pages = num_pages; p.total = total; p.batch = (int)batch; p.max_blocks = (int)max_blocks;
  p.heads = FastDiv((uint32_t)kv_heads); p.d[0] = (int)dk; p.d[1] = (int)dv; p.page_shift = page_shift_of(page_size);
  const int64_t sms = device_info().sm_count;
  // Few tokens: fewer a CTA, so that fewer rows follow one another, up to three CTAs an SM (us with 4 / 8 / 16, 8 heads: 64 tokens
  // 2.5 / - / 4.3, 1000 2.9 / - / 4.5, 2000 4.5 / 3.8 / 4.5, 3200 - / 4.5 / 5.5, 4000 5.6 / 6.5 / 5.6).
  p.tokens = total <= 12 * sms ? 4 : total <= 24 * sms ? 8 : kGatherTokens;
  const unsigned ctas = (unsigned)((total + p.tokens - 1) / p.tokens);
  const bool bf16 = dtype == UNIQL_BF16;
  auto kernel = dp == 128 ? (bf16 ? kv4_gather_kernel<128, true> : kv4_gather_kernel<128, false>)
                          : (bf16 ? kv4_gather_kernel<64, true> : kv4_gather_kernel<64, false>);
  return launch_pdl(kernel, ctas, kGatherThreads, 0, (cudaStream_t)stream, p);
}
