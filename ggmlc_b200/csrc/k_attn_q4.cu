// Attention over a KV cache held in 4 bits, rows of q taken one by one (decode).
//
// Row r sees n_r = min(pos_r + 1, max_kv) positions.  With S = scale * q K^T, the output is
// softmax(S) V, kept as a running maximum m, sum l and accumulator O per q head (fp32).
//
// Both products run on the tensor cores as mma.sync m16n8k16 f16 with fp32 accumulators, the
// cache as the 16-row operand A and the q heads of one KV head as the 8-column operand B, so up to
// 8 heads of a group share every decoded code: S^T [16 keys x 8 heads] = K q^T, then
// O^T [16 dims x 8 heads] += V^T P^T.  A warp walks keys in steps of 32 (64 at head_dim 64); lane
// (g, c) = (lane / 4, lane % 4) holds key g's words 4b + c of K, and dims [g hd/8, (g + 1) hd/8) of
// V for keys 2c, 2c + 1, 2c + 8, 2c + 9 of every group of 16: whole 32-bit words either way, decoded
// in registers.
//   A chunk's consecutive positions share the 8 columns where a KV head has at most 4 q heads.
//   K: codes enter the product as they are and the block scale multiplies the block's sum in fp32,
//      so K adds no rounding.  A nibble n becomes an f16 by OR with 0x6400: bits 0-3 give 1024 + n,
//      bits 4-7 give 1024 + 16 n.  16-bit q: q / 16 faces the latter, and the offsets leave through
//      one more product, (scales of the key) x -(1032 sum q_lo + 72 sum q_hi) of each block as three
//      f16 terms, so the codes are not touched again (a sum is of the order of 2^10 |q| before the
//      offsets cancel: 2e-5 of a score in fp32).
//      f32 q: the offsets are subtracted from the codes (exact), and q enters as the sum of two f16
//      terms (22 bits).
//   q is multiplied by a power of two per head, the largest element in [1, 2), so that bf16 and
//      f32 inputs fit f16; the factor returns in the softmax scale.
//   V: (n - 8) * d in f16, one rounding (16-bit types); f32: that and the exact remainder as a
//      second f16 term.  The rounding is 2^-12 of values whose codes are off by up to 2^-4 of their
//      block's extreme.  For f16 it is what is left above the rounding of the output (error against 64
//      bits 2.6e-4, the output alone 2.1e-4); the second term costs a row of 131071 positions 64 us
//      instead of 54.  Scales of positions past n_r are replaced by zero, and their scores by
//      -inf, by selection: what the memory holds there (NaN included) is never multiplied in.
//      Packed positions see different numbers of keys: a key that only some of them see and whose
//      V scale is no number gets scale zero, and the columns that see it get their NaN by addition.
//   P: exp2(s - m + 14) in f16 (two terms for f32 and f16 outputs); the factor 2^14 cancels in O / l and
//      keeps small probabilities out of f16's subnormals.  One term is enough for bf16, whose error is
//      1.6e-3 as the output's rounding alone makes; two cost 64 ragged rows 164 us instead of 151.
//      Whoever wants f32's arithmetic for 16-bit data passes q as f32 (227 us).
//
// Work split: a step is a run of kKeys keys of one row, KV head and up to 8 heads of its group; a
// segment is one CTA's run of steps of one row and head group, its 4 warps taking them in turn.
// The grid fills the machine once, and every CTA derives its segments from the rows' positions by
// itself.  Few rows: each row and head group is cut evenly into CTAs.  Many:
// the steps of all rows and head groups form one list, with kOverhead units in front of each group
// for what a segment costs besides its steps, and every CTA takes an equal range of it, so ragged
// rows balance.  A segment cut between CTAs leaves (m, l, O) in the workspace, at most two per CTA;
// the CTA that finishes last (a counter, reset on the way out) joins the parts in order, in runs of
// kFan and then the runs when there are more, so the result does not depend on which CTA that is.
// (One CTA reading all 54 parts of a 131071-position row took 19 us.)
// Data path: each warp owns a ring of stages that it keeps filled, across segments, with 16-byte
// cp.async (9 a lane and step at head_dim 128); page rows are contiguous, so one address serves a
// step, or one per 16 keys where a page ends inside a step.  (Bulk copies issued by one lane took
// 4 per warp and step; their operands cost a fifth of the loop's issue slots.)
// Bound: by issue slots.  A step of 32 keys at head_dim 128 is 737 warp instructions in bf16 (321 of
// them integer, 262 fp), at 2.6 a clock and SM: 64 rows of 1..16384 positions of 8 x 128 151 us (the
// bytes alone 93), one row of 131071 in f16 55 us (23).  Short rows by latency: one of 640 in f32 10.4
// us, of which an empty launch is 2.2.  (Calls queued one after the other, CUDA events.)
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "../../include/ggmlc_b200.h"
#include "common.h"
#include "kernels.h"
#include "kq4.cuh"
#include "kutil.cuh"

namespace gb {

namespace {

constexpr int kMaxRowsCall = 1024;
constexpr int kHeads = 8;        // q heads per item (MMA columns)
// what a segment costs besides its steps (its q, the join of its warps), in steps; and the fewest
// steps worth a CTA of their own
constexpr int kOverhead = 10;
constexpr int kMinSteps = 8;
constexpr int kFan = 8;         // parts joined by one CTA; more of them in two levels
constexpr float kPShift = 14.0f;
constexpr float kLog2e = 1.4426950408889634f;

// 4 consecutive outputs acc / l (zeros where nothing was seen)
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 acc, float l) {
    const float r = l != 0.0f ? 1.0f / l : 0.0f;
    const float v[4] = {acc.x * r, acc.y * r, acc.z * r, acc.w * r};
#pragma unroll
    for (int j = 0; j < 4; ++j) q4_put(p + j, v[j]);
}

// D += A B, m16n8k16, f16 operands, fp32 accumulators
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// D = A B
__device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t su32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
// 16 bytes from src + OFF to dst + DOFF in shared memory
template <int DOFF, int OFF>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src),
                 "n"(DOFF), "n"(OFF)
                 : "memory");
}
// compile-time loop: f(integral_constant 0 .. N - 1)
template <int N, class F>
__device__ __forceinline__ void unroll(F&& f) {
    if constexpr (N > 0) {
        unroll<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
// 16 bytes to shared memory, or 16 zero bytes (nothing is read) when !real
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(real ? 16 : 0)
                 : "memory");
}

// N 32-bit words from shared memory in the widest loads
template <int N>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *(const uint4*)(p + 4 * i);
            w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *(const uint2*)p;
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *(const uint32_t*)p;
    }
}

// shapes of one build: keys per step, ring stages, CTAs per SM
template <int HD, int PREC>
struct Shape {
    static constexpr int kKeys = HD == 64 ? 64 : 32;
    static constexpr int kStages = HD == 256 ? 2 : 3;
    // 12 warps an SM (registers) as 3 CTAs of 4; as 2 of 6 or 1 of 12 the joins of a CTA's warps
    // hold up more of them: 64 ragged rows of up to 16384 positions 150 / 166 / 200 us
    static constexpr int kWarps = 4;
    static constexpr int kCtas = HD == 256 ? 2 : 3;
    static constexpr int kBufs = 2;  // where the warps' outputs meet
    static constexpr int kCode = kKeys * HD / 2, kScale = kKeys * HD / 16;
    static constexpr int kStage = 2 * (kCode + kScale);
    static constexpr int kRing = kStage * kStages * kWarps;
    static constexpr int kPad = HD + 4;
    static constexpr int kSmem = kRing + kBufs * kHeads * kPad * 4;
};

// A row of work: one row of q, or a chunk's `pack` consecutive positions (heads of both as columns).
// keys that row r's position i sees; those of the row's last position
__device__ __forceinline__ int keys_seen(const AttnQ4Args& a, int64_t i) {
    return (int)min(kv_q4_pos(a.r, i) + 1, a.max_kv);
}
__device__ __forceinline__ int row_keys(const AttnQ4Args& a, int64_t r) {
    return keys_seen(a, min((r + 1) * a.pack, a.r.n) - 1);
}
// steps of a row: at least one, so that a row that sees nothing is written too
template <int KEYS>
__device__ __forceinline__ int row_steps(const AttnQ4Args& a, int64_t r) {
    const int n = row_keys(a, r);
    return n > 0 ? (int)(((int64_t)n + KEYS - 1) / KEYS) : 1;
}

// inclusive sum over the CTA of one value per thread
__device__ __forceinline__ long long cta_scan(long long v, long long* warp_sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += warp_sum[w];
    return v;
}

// one CTA's part of a row and head group: steps [begin, end) of its `steps`; hk, grp: KV head and
// which 8 of its q heads; at: the first unit of the row and head group, counted from the CTA's
// first; parts: CTAs it is cut into (one segment per CTA only)
struct Segment {
    int at, row, hk, grp, begin, end, steps, parts;
};

// CTAs of one launch: the machine filled once.  The workspace: 3 counters per CTA, then 4 partials
constexpr int kMaxCtas = 1024, kMaxCtasPerSm = 3;
constexpr int64_t kCounterBytes = 3 * kMaxCtas * 4;
static_assert(kCounterBytes <= GB_KV_Q4_WORK_ZEROED, "the counters are what callers zero");
constexpr int64_t partial_floats(int64_t hd) { return kHeads * (hd + 2); }

// whether this CTA is the last of n to arrive at the counter (which it then resets); what the
// others wrote before is visible to all its threads
__device__ __forceinline__ bool last_of(int* counter, int n, int* s_last) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        *s_last = atomicAdd(counter, 1) == n - 1;
        if (*s_last) *counter = 0;
    }
    __syncthreads();
    const bool last = *s_last;
    __syncthreads();
    if (last) __threadfence();
    return last;
}

// Joins parts first .. first + n - 1 in order, kFan at a time in flight, with a running maximum:
// the output (out(h): head h's HD values), or another partial `to`.
template <typename T, int HD, int kThreads, class At, class Out>
__device__ __forceinline__ void join(const At& at, int first, int n, int heads, const Out& out,
                                     float* to) {
    // groups of 4 dims a thread joins at once
    constexpr int kCols = kHeads * (HD / 4) > kThreads ? 2 : 1;
    const int cols = heads * (HD / 4);
#pragma unroll 1
    for (int e0 = threadIdx.x; e0 < cols; e0 += kThreads * kCols) {
        float4 acc[kCols];
        float m[kCols], l[kCols];
        int where[kCols], ml[kCols];
#pragma unroll
        for (int k = 0; k < kCols; ++k) {
            const int e = min(e0 + k * kThreads, cols - 1);
            where[k] = e * 4;
            ml[k] = kHeads * HD + 2 * (e / (HD / 4));
            acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            m[k] = -INFINITY;
            l[k] = 0.0f;
        }
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += kFan) {
            float4 v[kCols][kFan];
            float2 st[kCols][kFan];
#pragma unroll
            for (int i = 0; i < kFan; ++i) {
                const float* p = at(first + min(i0 + i, n - 1));
#pragma unroll
                for (int k = 0; k < kCols; ++k) {
                    st[k][i] = __ldcg((const float2*)(p + ml[k]));
                    v[k][i] = __ldcg((const float4*)(p + where[k]));
                }
            }
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                float x = m[k];
#pragma unroll
                for (int i = 0; i < kFan; ++i) x = fmaxf(x, st[k][i].x);
                const float ref = x == -INFINITY ? 0.0f : x;
                float w = ex2(m[k] - ref);
                m[k] = x;
                l[k] *= w;
                acc[k].x *= w, acc[k].y *= w, acc[k].z *= w, acc[k].w *= w;
#pragma unroll
                for (int i = 0; i < kFan; ++i) {
                    w = ex2(st[k][i].x - ref);
                    if (i0 + i < n) {
                        l[k] = fmaf(w, st[k][i].y, l[k]);
                        acc[k].x = fmaf(w, v[k][i].x, acc[k].x);
                        acc[k].y = fmaf(w, v[k][i].y, acc[k].y);
                        acc[k].z = fmaf(w, v[k][i].z, acc[k].z);
                        acc[k].w = fmaf(w, v[k][i].w, acc[k].w);
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kCols; ++k) {
            if (e0 + k * kThreads >= cols) break;
            if (to) {
                *(float4*)(to + where[k]) = acc[k];
                if (where[k] % HD == 0) *(float2*)(to + ml[k]) = make_float2(m[k], l[k]);
            } else {
                store4(out(where[k] / HD) + where[k] % HD, acc[k], l[k]);
            }
        }
    }
}

// PREC: 0 one f16 term everywhere (bf16), 1 two-term operands (f32), 2 two-term probabilities (f16).
// PACK: rows of work are several positions of a chunk (a.pack > 1)
template <typename T, int HD, int PREC, bool PACK>
__global__ void __launch_bounds__(Shape<HD, PREC>::kWarps * 32, Shape<HD, PREC>::kCtas)
    k_attn_q4(const __grid_constant__ AttnQ4Args a, int groups, int* counters, float* parts) {
    pdl_launch();
    pdl_wait();
    using S = Shape<HD, PREC>;
    constexpr int kWarps = S::kWarps, kThreads = kWarps * 32;
    constexpr int KEYS = S::kKeys;
    constexpr int NB = HD / 32;    // blocks per row
    constexpr int MT = HD / 16;    // 16-dim tiles of O^T
    constexpr int VW = HD / 64;    // V words per lane and key
    constexpr int NG = KEYS / 16;  // 16-key groups per step
    constexpr bool kExactQ = PREC == 1, kTwoP = PREC != 0;
    extern __shared__ __align__(128) uint8_t smem[];
    float* s_o = (float*)(smem + S::kRing);  // [kBufs][kHeads][kPad]
    __shared__ long long s_first[kMaxRowsCall + 1];  // steps before a row (times the head groups)
    __shared__ long long s_warp[kWarps];
    __shared__ float s_m[kWarps][kHeads], s_l[kWarps][kHeads];
    __shared__ int s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, c = lane & 3;
    const int rows = (int)((a.r.n + a.pack - 1) / a.pack);
    const int hgs = a.c.Hkv * groups;

    // ---- this CTA's part of the work.  s_first: sums over the rows before r, times the head groups,
    // of the rows' steps, or (one segment per CTA) of the CTAs they are cut into
    __shared__ int s_longest;  // the largest value of up to 32 rows
    auto prefix = [&](auto value) {
        if (rows <= 32) {
            if (warp == 0) {
                long long v = lane < rows ? value(lane) : 0;
                const int top = __reduce_max_sync(0xffffffffu, (int)v);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long u = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += u;
                }
                if (lane < rows) s_first[lane + 1] = v * hgs;
                if (lane == 0) s_longest = top;
            }
        } else {
            long long before = 0;
            for (int r0 = 0; r0 < rows; r0 += kThreads) {
                const int r = r0 + tid;
                const long long incl = before + cta_scan(r < rows ? value(r) : 0, s_warp);
                if (r < rows) s_first[r + 1] = incl * hgs;
                if (r0 + kThreads < rows) {
                    __syncthreads();
                    before = s_first[r0 + kThreads] / hgs;
                }
            }
        }
        if (tid == 0) {
            s_first[0] = 0;
            if (rows > 32) s_longest = 0;
        }
        __syncthreads();
    };
    prefix([&](int r) { return (long long)row_steps<KEYS>(a, r); });
    const long long steps_all = s_first[rows];
    const bool apart = 2 * (long long)rows * hgs <= gridDim.x;  // one segment per CTA
    long long per = 1, w0 = blockIdx.x;  // units per CTA; the CTA's first unit
    int range = 1;                       // units of this CTA
    long long budget = 0;
    if (apart) {
        // The machine filled once, but no CTA for less than kMinSteps, or one step a warp where that
        // leaves the longest row at most kFan parts, which one CTA joins.  Measured, f32: 640 positions
        // 11.4 us with 8 steps a CTA, 10.4 with 4 (1000 positions 12.0 and 10.6); 2000 positions 12.5 with
        // 8, 14.6 with 5 and two levels of joins; 200 positions 9.4 whole, 9.6 with 4.
        const int least = s_longest > kMinSteps && s_longest <= kWarps * kFan ? kWarps : kMinSteps;
        budget = max((long long)least, (steps_all - 1) / ((long long)gridDim.x - rows * hgs) + 1);
        __syncthreads();
        prefix([&](int r) { return (row_steps<KEYS>(a, r) + budget - 1) / budget; });
        if (w0 >= s_first[rows]) return;
    } else {
        const long long total = steps_all + (long long)rows * hgs * kOverhead;
        per = max((long long)kOverhead + kWarps, (total - 1) / gridDim.x + 1);
        w0 *= per;
        if (w0 >= total) return;
        range = (int)min(per, total - w0);
    }
    const int extra = apart ? 0 : kOverhead * hgs;  // units per row on top of s_first
    Segment first;
    first.row = 0;
    for (int hi = rows - 1; first.row < hi;) {  // the row of unit w0
        const int mid = (first.row + hi + 1) >> 1;
        if (s_first[mid] + (long long)mid * extra <= w0) first.row = mid; else hi = mid - 1;
    }
    {
        const long long in_row = w0 - s_first[first.row] - (long long)first.row * extra;
        first.steps = row_steps<KEYS>(a, first.row);
        // units of one head group, of which the first `lead` are no steps
        const int units = apart ? (int)((s_first[first.row + 1] - s_first[first.row]) / hgs)
                                : first.steps + kOverhead;
        const int hg = (int)(in_row / units), at = (int)(in_row - (long long)hg * units);
        first.hk = hg / groups;
        first.grp = hg - first.hk * groups;
        first.at = -at;
        if (apart) {
            first.begin = (int)((long long)first.steps * at / units);
            first.end = (int)((long long)first.steps * (at + 1) / units);
            first.parts = units;
        } else {
            first.begin = max(0, at - kOverhead);
            first.end = min(first.steps, at + range - kOverhead);
            first.parts = 0;
        }
    }
    auto advance = [&](Segment& sg) {  // the next segment; false past the CTA's range
        if (apart) return false;
        sg.at += sg.steps + kOverhead;
        if (sg.at + kOverhead >= range) return false;
        if (++sg.grp == groups) {
            sg.grp = 0;
            if (++sg.hk == a.c.Hkv) {
                sg.hk = 0;
                ++sg.row;
                sg.steps = (int)((s_first[sg.row + 1] - s_first[sg.row]) / hgs);
            }
        }
        sg.begin = 0;
        sg.end = min(sg.steps, range - sg.at - kOverhead);
        return true;
    };

    // ---- the warp's ring: copies run ahead of use, across segments
    const bool whole = !a.c.pages || a.c.page_len % KEYS == 0;  // no page ends inside a step
    const uint32_t page_len = (uint32_t)a.c.page_len;
    const int64_t page_stride = a.c.Hkv * a.c.page_bytes, scales = (int64_t)page_len * (HD / 2);
    Segment ps = first;  // segment and step of the next copy
    int pstep = ps.begin + warp, pn, pslot;
    const int32_t* plist;  // the sequence's pages
    int64_t phead;         // the head's place in a page
    auto locate = [&]() {
        const int64_t slot = kv_q4_slot(a.r, (int64_t)ps.row * a.pack);
        const bool in = slot >= 0 && slot < a.c.n_slots;
        pn = in ? row_keys(a, ps.row) : 0;  // a slot outside the cache has no pages
        pslot = in ? (int)slot : 0;
        plist = a.c.pages + (int64_t)pslot * a.c.per_slot;
        phead = ps.hk * a.c.page_bytes;
    };
    locate();
    bool more = true;
    int pstage = 0, stage = 0;  // ring places of the next copy and the next use
    uint32_t oks = 0;           // per ring place: 16-key groups that have a page
    auto issue = [&]() {  // requests the next step; an empty group once the range is exhausted
        while (more && pstep >= ps.end) {
            more = advance(ps);
            if (more) locate();
            pstep = ps.begin + warp;
        }
        if (more) {
            const int t0 = pstep * KEYS;
            int left = pn - t0;  // rows past it are not read: zeros
            const uint32_t st = su32(smem + (warp * S::kStages + pstage) * S::kStage) + lane * 16;
            uint32_t ok = 0;
            constexpr int kRowB = HD / 2, kRowS = HD / 16;
            constexpr int kScaleChunks = 2 * S::kScale / 16;  // of both K and V
            static_assert(kScaleChunks == 32 || kScaleChunks == 64, "one or two a lane");
            const int row0 = lane * 16 / kRowB;               // row of the lane's first code chunk
            if (whole) {
                int64_t prow = t0;
                int pg = pslot;
                if (left > 0 && a.c.pages) {
                    const uint32_t i =
                        a.shift >= 0 ? (uint32_t)t0 >> a.shift : (uint32_t)t0 / page_len;
                    prow = (uint32_t)t0 - i * page_len;
                    pg = plist[i];
                    if (pg < 0 || pg >= a.c.n_pages) left = 0;
                }
                ok = left > 0 ? (1u << NG) - 1 : 0;
                const int64_t base = pg * page_stride + phead;
                const int64_t code = base + prow * kRowB + lane * 16;
                const uint8_t *kp = a.c.k + code, *vp = a.c.v + code;
                // lanes below kScale / 16 copy K scales, the others V scales
                const int at = lane * 16 % S::kScale;
                const uint8_t* sp = (lane * 16 < S::kScale ? a.c.k : a.c.v) + base + scales +
                                    prow * kRowS + at;
                if (left >= KEYS) {
                    unroll<S::kCode / 512>([&](auto i) {
                        copy16<i * 512, i * 512>(st, kp);
                        copy16<S::kCode + i * 512, i * 512>(st, vp);
                    });
                    copy16<2 * S::kCode, 0>(st, sp);
                    if constexpr (kScaleChunks > 32)  // kScale == 512: K above, V here
                        copy16<2 * S::kCode + 512, 0>(st, a.c.v + (sp - a.c.k));
                } else {
#pragma unroll
                    for (int i = 0; i < S::kCode / 512; ++i) {
                        const bool real = row0 + i * (512 / kRowB) < left;
                        copy16(st + i * 512, kp + i * 512, real);
                        copy16(st + S::kCode + i * 512, vp + i * 512, real);
                    }
                    copy16(st + 2 * S::kCode, sp, at / kRowS < left);
                    if constexpr (kScaleChunks > 32)
                        copy16(st + 2 * S::kCode + 512, a.c.v + (sp - a.c.k), at / kRowS < left);
                }
            } else {
                int64_t base[NG];
                int64_t prow[NG];
#pragma unroll
                for (int q = 0; q < NG; ++q) {
                    const uint32_t t = t0 + q * 16, i = t / page_len;
                    int pg = -1;
                    if (q * 16 < left) pg = plist[i];
                    const bool in = pg >= 0 && pg < a.c.n_pages;
                    ok |= (uint32_t)in << q;
                    base[q] = (in ? pg : 0) * page_stride + phead;
                    prow[q] = in ? t - i * page_len : 0;  // 32-bit remainder
                }
#pragma unroll
                for (int i = 0; i < S::kCode / 512; ++i) {
                    const int q = i * 512 / (16 * kRowB);  // 512 bytes lie in one group
                    const int64_t code =
                        base[q] + prow[q] * kRowB + (i * 512 - q * 16 * kRowB) + lane * 16;
                    const bool real = (ok >> q & 1) && row0 + i * (512 / kRowB) < left;
                    copy16(st + i * 512, a.c.k + code, real);
                    copy16(st + S::kCode + i * 512, a.c.v + code, real);
                }
#pragma unroll
                for (int i = 0; i < kScaleChunks; i += 32) {
                    const int at = (lane + i) * 16 % S::kScale, q = at / (16 * kRowS);
                    int64_t b = base[0] + prow[0] * kRowS;
#pragma unroll
                    for (int j = 1; j < NG; ++j)
                        if (q == j) b = base[j] + prow[j] * kRowS;
                    const uint8_t* pool = (lane + i) * 16 < S::kScale ? a.c.k : a.c.v;
                    copy16(st + 2 * S::kCode + i * 16, pool + b + scales + at - q * 16 * kRowS,
                           (ok >> q & 1) && at / kRowS < left);
                }
            }
            oks = (oks & ~(((1u << NG) - 1) << (pstage * NG))) | ok << (pstage * NG);
            if (++pstage == S::kStages) pstage = 0;
            pstep += kWarps;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");  // empty past the range
    };
#pragma unroll 1
    for (int i = 0; i < S::kStages; ++i) issue();

    const int Hq = a.Hq, rk = Hq / a.c.Hkv;
    Segment sg = first;
    do {
        // the segment's columns: up to 8 heads of a row, or those of its packed positions in turn
        const int64_t i0 = PACK ? (int64_t)sg.row * a.pack : sg.row;
        const int heads = PACK ? (int)min((int64_t)a.pack, a.r.n - i0) * rk
                               : min(kHeads, rk - sg.grp * kHeads);
        auto position = [&](int col) { return i0 + (PACK ? col / rk : 0); };
        auto head = [&](int col) {
            return sg.hk * rk + (PACK ? col % rk : sg.grp * kHeads + col);
        };
        auto out = [&](int col) { return (T*)a.o + (position(col) * Hq + head(col)) * HD; };
        const int n = row_keys(a, sg.row), n_first = PACK ? keys_seen(a, i0) : n;
        const int n0 = PACK ? keys_seen(a, min(position(2 * c), a.r.n - 1)) : n;
        const int n1 = PACK ? keys_seen(a, min(position(2 * c + 1), a.r.n - 1)) : n;

        // ---- q fragments: B operand, lane (g, c) holds dims 32b + 8c + j of head g
        uint32_t qh[NB][4], ql[kExactQ ? NB : 1][4];
        uint32_t off[kExactQ ? 1 : NB / 2];  // offsets of the block sums (B operand, see below)
        float qs;                            // softmax scale of head g in powers of two
        {
            const T* qp = (const T*)a.q;
            if (g < heads) qp += position(g) * a.q_row + (int64_t)head(g) * a.q_head;
            float x[NB][8], big = 0.0f, bad = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const T* p = qp + 32 * b + 8 * c;
                if (g >= heads) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[b][j] = 0.0f;
                } else if (a.q_vec) {
                    constexpr int N = 16 / sizeof(T);
#pragma unroll
                    for (int j = 0; j < 8; j += N) {
                        const uint4 raw = *(const uint4*)(p + j);
                        const T* e = (const T*)&raw;
#pragma unroll
                        for (int i = 0; i < N; ++i) x[b][j + i] = q4_to_f(e[i]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[b][j] = q4_to_f(p[j]);
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    big = fmaxf(big, fabsf(x[b][j]));
                    bad = fmaf(x[b][j], 0.0f, bad);  // NaN once an element is not finite
                }
            bad += __shfl_xor_sync(0xffffffffu, bad, 1);
            bad += __shfl_xor_sync(0xffffffffu, bad, 2);
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // 2^e with big / 2^e in [1, 2).  A head with an infinity or a NaN is NaN throughout: it has
            // NaN scores where it sees a key, and its masked scores stay -inf
            const int e = min(max((int)(__float_as_uint(big) >> 23) - 127, -126), 126);
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            float down = __uint_as_float((uint32_t)(127 - e) << 23);
            // a negative scale moves into q, a zero one becomes too small to tell scores apart: qs is
            // positive, so the largest raw sum is the largest score
            qs = fmaxf(fabsf(a.scale) * kLog2e * up, 1e-30f);
            if (a.scale < 0.0f) down = -down;
            auto pack = [&](float u, float v) { return h2u(__floats2half2_rn(u, v)); };
            float term[2];  // off of blocks b - 1, b: the c-th f16 term
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[b][j] = fmaf(x[b][j], down, bad);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float u = x[b][j], v = x[b][j + 4];
                    if constexpr (kExactQ) {
                        qh[b][j] = pack(u, v);
                        const float2 r = __half22float2(u2h(qh[b][j]));
                        ql[b][j] = pack(u - r.x, v - r.y);
                    } else if (j & 1) {
                        qh[b][j] = pack(u * 0.0625f, v * 0.0625f);
                        const float2 r = __half22float2(u2h(qh[b][j]));
                        s1 += r.x + r.y;
                    } else {
                        qh[b][j] = pack(u, v);
                        const float2 r = __half22float2(u2h(qh[b][j]));
                        s0 += r.x + r.y;
                    }
                }
                if constexpr (!kExactQ) {
                    float s = -(1032.0f * s0 + 1152.0f * s1);  // 72 q = 1152 (q / 16)
                    s += __shfl_xor_sync(0xffffffffu, s, 1);
                    s += __shfl_xor_sync(0xffffffffu, s, 2);
                    // s as three f16 terms (33 bits); lane c keeps the c-th, lane 3 none
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        const float t = __half2float(__float2half_rn(s));
                        if (i == c) term[b & 1] = t;
                        s -= t;
                    }
                    if (c == 3) term[b & 1] = 0.0f;
                    if (b & 1) off[b / 2] = pack(term[0], term[1]);
                }
            }
        }
        const float qs0 = __shfl_sync(0xffffffffu, qs, 8 * c);
        const float qs1 = __shfl_sync(0xffffffffu, qs, 8 * c + 4);

        float o[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

#pragma unroll 1
        for (int step = sg.begin + warp; step < sg.end; step += kWarps) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            __syncwarp();  // every lane's copies of this stage have landed
            uint8_t* st = smem + (warp * S::kStages + stage) * S::kStage;
            const uint32_t ok = oks >> (stage * NG) & ((1u << NG) - 1);
            const int valid = n - step * KEYS;  // < 1 for a row that sees nothing
            const bool all = n_first - step * KEYS >= KEYS && ok == (1u << NG) - 1;
            float s[NG][4];
#pragma unroll
            for (int q = 0; q < NG; ++q) {
                uint32_t w0_[NB], w1_[NB], d0_[NB / 2], d1_[NB / 2];
                const uint8_t* kp = st + (q * 16 + g) * (HD / 2) + c * (NB * 4);
                const uint8_t* kd = st + 2 * S::kCode + (q * 16 + g) * (HD / 16);
                lds<NB>(kp, w0_);
                lds<NB>(kp + 8 * (HD / 2), w1_);
                lds<NB / 2>(kd, d0_);
                lds<NB / 2>(kd + 8 * (HD / 16), d1_);
                if constexpr (kExactQ) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[q][j] = 0.0f;
                } else {
                    // sum over blocks of scale * offset: k-slots 2c, 2c + 1 (and + 8) are a pair of
                    // blocks, for the c-th term of their offsets, so A is the scales as they lie
#pragma unroll
                    for (int b = 0; b < NB / 2; b += 2) {
                        const bool two = b + 1 < NB / 2;
                        const uint32_t av[4] = {d0_[b], d1_[b], two ? d0_[b + two] : 0u,
                                                two ? d1_[b + two] : 0u};
                        if (b == 0)
                            mma0(s[q], av, off[b], two ? off[b + two] : 0u);
                        else
                            mma(s[q], av, off[b], two ? off[b + two] : 0u);
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float acc[4];
                    uint32_t f0[4], f1[4];
                    if constexpr (kExactQ) {
                        __half2 u0[4], u1[4];
                        codes(w0_[b], u0);
                        codes(w1_[b], u1);
#pragma unroll
                        for (int j = 0; j < 4; ++j) f0[j] = h2u(u0[j]), f1[j] = h2u(u1[j]);
                    } else {
                        nibbles(w0_[b], f0);
                        nibbles(w1_[b], f1);
                    }
                    const uint32_t a0[4] = {f0[0], f1[0], f0[1], f1[1]};
                    const uint32_t a1[4] = {f0[2], f1[2], f0[3], f1[3]};
                    if constexpr (kExactQ) {
                        mma0(acc, a0, ql[b][0], ql[b][1]);
                        mma(acc, a1, ql[b][2], ql[b][3]);
                        mma(acc, a0, qh[b][0], qh[b][1]);
                    } else {
                        mma0(acc, a0, qh[b][0], qh[b][1]);
                    }
                    mma(acc, a1, qh[b][2], qh[b][3]);
                    const __half2 e0 = u2h(d0_[b / 2]), e1 = u2h(d1_[b / 2]);
                    const float k0 = b & 1 ? __high2float(e0) : __low2float(e0);
                    const float k1 = b & 1 ? __high2float(e1) : __low2float(e1);
                    s[q][0] = fmaf(acc[0], k0, s[q][0]);
                    s[q][1] = fmaf(acc[1], k0, s[q][1]);
                    s[q][2] = fmaf(acc[2], k1, s[q][2]);
                    s[q][3] = fmaf(acc[3], k1, s[q][3]);
                }
                if (!all) {  // keys past the end or on no page
                    const bool pg = ok >> q & 1;
                    const int key = step * KEYS + q * 16 + g;
                    if (!pg || key >= n0) s[q][0] = -INFINITY;
                    if (!pg || key >= n1) s[q][1] = -INFINITY;
                    if (!pg || key + 8 >= n0) s[q][2] = -INFINITY;
                    if (!pg || key + 8 >= n1) s[q][3] = -INFINITY;
                }
            }
            float x0 = fmaxf(s[0][0], s[0][2]), x1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
            for (int q = 1; q < NG; ++q) {
                x0 = fmaxf(x0, fmaxf(s[q][0], s[q][2]));
                x1 = fmaxf(x1, fmaxf(s[q][1], s[q][3]));
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            x0 = fmaxf(m0, x0 * qs0);
            x1 = fmaxf(m1, x1 * qs1);
            // nothing seen yet: any finite reference keeps exp2(-inf) = 0
            const float r0 = x0 == -INFINITY ? 0.0f : x0, r1 = x1 == -INFINITY ? 0.0f : x1;
            if (__any_sync(0xffffffffu, x0 != m0 || x1 != m1)) {
                const float k0 = ex2(m0 - r0), k1 = ex2(m1 - r1);
                l0 *= k0, l1 *= k1;
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    o[i][0] *= k0, o[i][1] *= k1, o[i][2] *= k0, o[i][3] *= k1;
                m0 = x0, m1 = x1;
            }
            int bad_key = INT_MAX;  // PACK: the first such key of the lane's block
            bool any_bad = false;
            if (PACK && step * KEYS + KEYS > n_first) {
                // at most 7 keys; lanes c of a quad look at two each
                const int k0 = max(n_first - step * KEYS, 0) + c, end = min(valid, KEYS);
                uint16_t* sc = (uint16_t*)(st + 2 * S::kCode + S::kScale) + g * (HD / 8) / 32;
                const bool b0 = k0 < end && bad_scales(sc[k0 * NB]);
                const bool b1 = k0 + 4 < end && bad_scales(sc[(k0 + 4) * NB]);
                any_bad = __any_sync(0xffffffffu, b0 || b1);  // every lane has read
                if (any_bad) {
                    if (b0) sc[k0 * NB] = 0;
                    if (b1) sc[(k0 + 4) * NB] = 0;
                    bad_key = b0 ? step * KEYS + k0 : b1 ? step * KEYS + k0 + 4 : INT_MAX;
                    bad_key = min(bad_key, __shfl_xor_sync(0xffffffffu, bad_key, 1));
                    bad_key = min(bad_key, __shfl_xor_sync(0xffffffffu, bad_key, 2));
                    __syncwarp();
                }
            }
#pragma unroll
            for (int q = 0; q < NG; ++q) {
                float p[4];
                p[0] = ex2(fmaf(s[q][0], qs0, kPShift - r0));
                p[1] = ex2(fmaf(s[q][1], qs1, kPShift - r1));
                p[2] = ex2(fmaf(s[q][2], qs0, kPShift - r0));
                p[3] = ex2(fmaf(s[q][3], qs1, kPShift - r1));
                l0 += p[0] + p[2];
                l1 += p[1] + p[3];
                const __half2 ph0 = __floats2half2_rn(p[0], p[1]), ph1 = __floats2half2_rn(p[2], p[3]);
                const uint32_t b0 = transpose8x8(h2u(ph0)), b1 = transpose8x8(h2u(ph1));
                uint32_t bl0 = 0, bl1 = 0;
                if constexpr (kTwoP) {
                    const float2 f0 = __half22float2(ph0), f1 = __half22float2(ph1);
                    bl0 = transpose8x8(h2u(__floats2half2_rn(p[0] - f0.x, p[1] - f0.y)));
                    bl1 = transpose8x8(h2u(__floats2half2_rn(p[2] - f1.x, p[3] - f1.y)));
                }
                // V: keys 2c, 2c + 1 (pair 0) and 2c + 8, 2c + 9 (pair 1)
                uint32_t w[4][VW];
                uint32_t dv[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = q * 16 + 2 * c + (e & 1) + 8 * (e >> 1);
                    lds<VW>(st + S::kCode + key * (HD / 2) + g * (VW * 4), w[e]);
                    dv[e] = *(const uint16_t*)(st + 2 * S::kCode + S::kScale + key * (HD / 16) +
                                               (g * (HD / 8) / 32) * 2);
                    if (!all && !((ok >> q & 1) && key < valid)) dv[e] = 0;
                }
                const __half2 d01 = u2h(__byte_perm(dv[0], dv[1], 0x5410));
                const __half2 d23 = u2h(__byte_perm(dv[2], dv[3], 0x5410));
#pragma unroll
                for (int i = 0; i < VW; ++i) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {  // dims 0-3, 4-7 of the word
                        const unsigned sel = hf ? 0x7632u : 0x5410u;
                        __half2 u0[4], u1[4];
                        codes(__byte_perm(w[0][i], w[1][i], sel), u0);
                        codes(__byte_perm(w[2][i], w[3][i], sel), u1);
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            const __half2 e0 = __hmul2(u0[j], d01), e1 = __hmul2(u0[j + 1], d01);
                            const __half2 e2 = __hmul2(u1[j], d23), e3 = __hmul2(u1[j + 1], d23);
                            const uint32_t av[4] = {h2u(e0), h2u(e1), h2u(e2), h2u(e3)};
                            float(&acc)[4] = o[i * 4 + hf * 2 + j / 2];
                            if constexpr (kExactQ) {
                                const uint32_t al[4] = {
                                    h2u(__hfma2(u0[j], d01, __hneg2(e0))),
                                    h2u(__hfma2(u0[j + 1], d01, __hneg2(e1))),
                                    h2u(__hfma2(u1[j], d23, __hneg2(e2))),
                                    h2u(__hfma2(u1[j + 1], d23, __hneg2(e3)))};
                                // the tensor cores' fp32 sums truncate: over a long row the same way every
                                // time (1.2e-5 of the output at 14676 positions), so 16 keys at most
                                // are summed there and the rest rounds to nearest
                                float part[4];
                                mma0(part, al, b0, b1);
                                mma(part, av, bl0, bl1);
                                mma(part, av, b0, b1);
#pragma unroll
                                for (int k = 0; k < 4; ++k) acc[k] += part[k];
                            } else {
                                if constexpr (kTwoP) mma(acc, av, bl0, bl1);
                                mma(acc, av, b0, b1);
                            }
                        }
                    }
                }
            }
            if (PACK && any_bad) {
                const float nan = __int_as_float(0x7FFFFFFF);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (bad_key < n0) o[i][0] = nan, o[i][2] = nan;
                    if (bad_key < n1) o[i][1] = nan, o[i][3] = nan;
                }
            }
            if (++stage == S::kStages) stage = 0;
            __syncwarp();  // every lane has read the stage: it may be filled again
            issue();
        }

        // ---- the warps' states meet in shared memory: the first kBufs store, the others add
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        __syncthreads();  // the previous segment's reads are done
        if (g == 0) {
            s_m[warp][2 * c] = m0, s_m[warp][2 * c + 1] = m1;
            s_l[warp][2 * c] = l0, s_l[warp][2 * c + 1] = l1;
        }
        __syncthreads();
        float x0 = s_m[0][2 * c], x1 = s_m[0][2 * c + 1];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            x0 = fmaxf(x0, s_m[w][2 * c]);
            x1 = fmaxf(x1, s_m[w][2 * c + 1]);
        }
        const float f0 = ex2(m0 - (x0 == -INFINITY ? 0.0f : x0));
        const float f1 = ex2(m1 - (x1 == -INFINITY ? 0.0f : x1));
        for (int turn = 0; turn < (kWarps + S::kBufs - 1) / S::kBufs; ++turn) {
            if (warp / S::kBufs == turn) {
                float* d0 = s_o + (warp % S::kBufs * kHeads + 2 * c) * S::kPad + g * (HD / 8);
                float* d1 = d0 + S::kPad;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    float2 u = make_float2(o[i][0] * f0, o[i][2] * f0);
                    float2 v = make_float2(o[i][1] * f1, o[i][3] * f1);
                    if (turn) {
                        const float2 pu = *(const float2*)(d0 + 2 * i), pv = *(const float2*)(d1 + 2 * i);
                        u.x += pu.x, u.y += pu.y, v.x += pv.x, v.y += pv.y;
                    }
                    *(float2*)(d0 + 2 * i) = u;
                    *(float2*)(d1 + 2 * i) = v;
                }
            }
            __syncthreads();
        }
        // which CTAs hold parts of this row and head group
        const bool cut = sg.begin != 0 || sg.end != sg.steps;
        const long long unit0 = w0 + sg.at;
        const int cta0 = apart ? (int)unit0 : (int)((unit0 + kOverhead) / per);
        const int cta1 = apart ? cta0 + sg.parts - 1
                               : (int)((unit0 + kOverhead + sg.steps - 1) / per);
        // a CTA leaves the segment its range begins with in slot 0, the one it ends with in slot 1
        float* part = parts + (2 * (int64_t)blockIdx.x + (sg.at > 0)) * partial_floats(HD);
        for (int e = tid; e < heads * (HD / 4); e += kThreads) {
            const int h = e / (HD / 4), dim = e % (HD / 4) * 4;
            float m = s_m[0][h], l = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w][h]);
            const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) l += ex2(s_m[w][h] - ref) * s_l[w][h];
            float4 acc = *(const float4*)(s_o + h * S::kPad + dim);
#pragma unroll
            for (int i = 1; i < S::kBufs; ++i) {
                const float4 v = *(const float4*)(s_o + (i * kHeads + h) * S::kPad + dim);
                acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            }
            if (!cut) {
                store4(out(h) + dim, acc, l);
            } else {
                *(float4*)(part + h * HD + dim) = acc;
                if (dim == 0) {
                    part[kHeads * HD + 2 * h] = m;
                    part[kHeads * HD + 2 * h + 1] = l;
                }
            }
        }
        if (cut) {
            const int n_parts = cta1 - cta0 + 1, mine = blockIdx.x - cta0;
            const auto at = [&](int slot) { return parts + slot * partial_floats(HD); };
            const auto leaf = [&](int j) {
                return at(2 * (cta0 + j) + (j == 0 && unit0 > cta0 * per));
            };
            // joins of kFan parts, above them their own partials: one per CTA and kind (the first
            // run of a segment, or a later one), behind the leaves
            const auto inner = [&](int run) {
                return at(2 * (gridDim.x + cta0 + run * kFan) + (run > 0));
            };
            const int run = mine / kFan, runs = (n_parts + kFan - 1) / kFan;
            int* count = counters + (run > 0) * kMaxCtas + cta0 + run * kFan;
            if (last_of(count, min(kFan, n_parts - run * kFan), &s_last)) {
                if (runs == 1) {
                    join<T, HD, kThreads>(leaf, 0, n_parts, heads, out, nullptr);
                } else {
                    join<T, HD, kThreads>(leaf, run * kFan, min(kFan, n_parts - run * kFan), heads, out,
                                inner(run));
                    if (last_of(counters + 2 * kMaxCtas + cta0, runs, &s_last))
                        join<T, HD, kThreads>(inner, 0, runs, heads, out, nullptr);
                }
            }
        }
    } while (advance(sg));
}

int64_t head_groups(int64_t Hq, int64_t Hkv) {
    return Hkv * ((Hq / Hkv + kHeads - 1) / kHeads);
}


template <typename T, int HD, int PREC, bool PACK>
void launch_t(const AttnQ4Args& a, cudaStream_t st) {
    using S = Shape<HD, PREC>;
    static_assert(S::kCtas <= kMaxCtasPerSm, "workspace");
    int dev = 0;
    GB_CUDA(cudaGetDevice(&dev));
    static std::atomic<bool> ready[64];
    if (dev >= 64 || !ready[dev]) {
        GB_CUDA(cudaFuncSetAttribute(k_attn_q4<T, HD, PREC, PACK>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        if (dev < 64) ready[dev] = true;
    }
    const int64_t hg = head_groups(a.Hq, a.c.Hkv);
    // no more CTAs than the rows can give work to; the list itself is made on the device
    const int64_t steps = std::max<int64_t>(1, (a.max_kv + S::kKeys - 1) / S::kKeys);
    const int64_t most =
        (a.r.n + a.pack - 1) / a.pack * hg * std::max<int64_t>(2, (steps + S::kWarps - 1) / S::kWarps + 1);
    const int grid = (int)std::min<int64_t>(most, (int64_t)sm_count(dev) * S::kCtas);
    int* counters = (int*)a.work;
    float* parts = (float*)((char*)a.work + kCounterBytes);
    AttnQ4Args b = a;
    b.shift = kv_q4_shift(a.c);
    b.q_vec = kv_q4_vectors(a);
    launch_pdl(k_attn_q4<T, HD, PREC, PACK>, grid, dim3(S::kWarps * 32), S::kSmem, st, b,
               (int)(hg / a.c.Hkv), counters, parts);
}

template <typename T, int PREC, bool PACK>
void launch_hd(const AttnQ4Args& a, cudaStream_t st) {
    switch (a.c.hd) {
        case 64: launch_t<T, 64, PREC, PACK>(a, st); break;
        case 128: launch_t<T, 128, PREC, PACK>(a, st); break;
        case 256: launch_t<T, 256, PREC, PACK>(a, st); break;
        default: GB_CHECK(false, "attn_q4: head_dim must be 64, 128 or 256");
    }
}

template <typename T, int PREC>
void launch_rows(const AttnQ4Args& a, cudaStream_t st) {
    if (a.pack > 1)
        launch_hd<T, PREC, true>(a, st);
    else
        launch_hd<T, PREC, false>(a, st);
}

}  // namespace

bool attn_q4_head_dim(int64_t hd) { return hd == 64 || hd == 128 || hd == 256; }

size_t attn_q4_parts_offset() { return kCounterBytes; }

size_t attn_q4_workspace(int64_t hd, bool chunks) {
    int dev = 0;
    GB_CUDA(cudaGetDevice(&dev));
    const int64_t ctas = (int64_t)sm_count(dev) * kMaxCtasPerSm;
    GB_CHECK(ctas <= kMaxCtas, "attn_q4: more SMs than the counters are made for");
    const size_t rows = (size_t)(4 * ctas * partial_floats(hd) * 4);
    return (size_t)kCounterBytes + std::max(rows, chunks ? attn_q4_tc_parts(hd) : 0);
}

void launch_attn_q4(const AttnQ4Args& args, cudaStream_t st) {
    const size_t es = args.type == kTypeF32 ? 4 : 2;
    // the 8 columns take several positions of a chunk where a KV head has at most 4 q heads
    const int64_t rk = args.Hq / args.c.Hkv;
    const bool chunk = args.r.n > 1 && !args.r.pos && !args.r.slot;
    const int pack = chunk && rk <= kHeads / 2 ? (int)(kHeads / rk) : 1;
    if (chunk && attn_q4_tc_fits(args)) {
        // A chunk by rows: each row and head group is a segment of steps.  As many segments as CTAs
        // or fewer: 5 us and 1.15 ns a step of 32 keys.  More: 9 us, and 1.05 ns for every step (half at
        // head_dim 64) and kOverhead more a segment.  By tiles: what the tile kernel's plan says.
        // Measured, bf16, rows / tiles: 32 heads of 128, 17 tokens at 1000 13.5 / 14.5, 100 at 0 16.0 /
        // 8.9; 9 heads of 64, 17 at 8000 15.0 / 20.6, 256 at 0 13.3 / 8.9.
        int dev = 0;
        GB_CUDA(cudaGetDevice(&dev));
        const double segments =
            (double)((args.r.n + pack - 1) / pack) * (double)head_groups(args.Hq, args.c.Hkv);
        const double most = (double)((args.max_kv + 31) / 32);
        const double mean =  // the chunk's middle row, as far as the host knows
            args.r.step_pos ? most : std::min(most, (double)(args.r.pos0 + args.r.n / 2 + 31) / 32);
        const double rows_us =
            2 * segments <= sm_count(dev) * Shape<128, 0>::kCtas
                ? 5.0 + 1.15e-3 * segments * most
                : 9.0 + 1.05e-3 * segments * (mean * (double)args.c.hd / 128 + kOverhead);
        if (attn_q4_tc_us(args) < rows_us) {
            launch_attn_q4_tc(args, st);
            return;
        }
    }
    const int64_t call = (int64_t)kMaxRowsCall * pack;
    for (int64_t r0 = 0; r0 < args.r.n; r0 += call) {
        AttnQ4Args a = args;
        a.pack = pack;
        a.r.n = std::min(call, args.r.n - r0);
        if (a.r.pos) a.r.pos += r0; else a.r.pos0 += r0;
        if (a.r.slot) a.r.slot += r0;
        a.q = (const char*)args.q + r0 * args.q_row * es;
        a.o = (char*)args.o + r0 * args.Hq * args.c.hd * es;
        switch (a.type) {
            case kTypeF32: launch_rows<float, 1>(a, st); break;
            case kTypeF16: launch_rows<__half, 2>(a, st); break;
            case kTypeBF16: launch_rows<__nv_bfloat16, 0>(a, st); break;
            default: GB_CHECK(false, "attn_q4: type must be f32, f16 or bf16");
        }
    }
    GB_CUDA(cudaGetLastError());
}

}  // namespace gb
