// Attention of a chunk (consecutive positions of one sequence, causal) over a KV cache held in 4
// bits, on the 5th-generation tensor cores: f16 and bf16 q, and f32 q of the engine's prefill
// (fast_f32), head_dim 64 and 128.
//
// A CTA takes two tiles of 128 q rows of one KV head, a row being a (position, head of the group)
// pair, and walks the keys in tiles of 128: S = Q K^T and O += P V as tcgen05.mma kind::f16 with
// fp32 accumulators in tensor memory (S and O of both tiles: 512 columns at head_dim 128).  S is
// made and used in halves of 64 keys, each its own buffer: the next scores of one half are computed
// while the softmax works on the other.
// Sharing one decoded K and V tile between 256 rows keeps the decode at a quarter of the
// instructions; two tiles let the softmax of one run under the products of the other.
//   K, V: (code - 8) * scale in f16, one rounding; for f16 calls K as the sum of two f16 terms, which
//   is exact (Q once more).  Measured at 333 tokens at 1999: 68 -> 83 us, and the error against 64
//   bits from 3.3e-4 to 2.6e-4 where rounding the output alone makes 2.1e-4.  V's second term has no
//   room in shared memory beside two tiles of Q (two stages of K and of V and K's second terms fill it).
//   bf16 calls: 1.68e-3, where rounding the output makes 1.66e-3; with f16's terms 2048 tokens at 14336
//   take 913 us instead of 565.  The engine's f32: 3.3e-4, of the size of what its prefill over an f16
//   cache rounds; 512 tokens at 0 take 20 us, with the rows kernel's 22 bits (3e-7) 65.
//   V of a key that only some rows of the CTA see must not reach the others through 0 x NaN: there a
//   scale that is no number is decoded as zero, and the first such key of each block of 32 dims kept;
//   rows that see it get NaN in the block when they are written.
//   q: f16 after a power of two per row, the largest element in [1, 2) (exact for bf16 but for
//   elements 2^-14 below it); the factor returns in the softmax scale.
//   P: exp2(s - m + 7) in f16, for f16 and f32 outputs as the sum of two f16 terms (V once more).  m is a
//   running maximum that is renewed only when a P would pass 2^15 (f16 holds 2^16): the scores are
//   read once, and O is rarely rescaled.
// Operands: all K-major with the 128-byte swizzle.  Q and K rows hold the 8 dims of a word in the
// order the nibbles come out of it (0 4 1 5 2 6 3 7), the same for both; V is transposed while it is
// decoded: the 16-bit halves of two keys' words are joined before the nibbles are spread, so a pair
// of keys of one dim comes out as an f16 pair.  P is read from tensor memory, written in place of S.
// Warps (20, one CTA per SM, registers split between the groups of 4):
//   0-3, 4-7  softmax of tile 0, 1: a thread owns a row (its tensor-memory lane), so its maximum and
//             sum need no exchange; they also load Q and write the output;
//   8-11      decode K tiles, 12-15 V tiles from global memory (the next tile's words are requested
//             before the current one is decoded), two stages each
//             (one for K's second terms, given back by halves);
//   16        issues the products, PV(j) then QK(j + 1) for each half and tile, and owns the tensor
//             memory (17-19 idle).
// Bound: at head_dim 128 a key tile costs 2048 clocks of tensor work (4 products of 128^3 at 4096
// multiply-adds a clock) and 2048 of exponentials (16 a clock), overlapped.
// Measured (bf16): 2048 tokens at 14336 of 32 heads 565 us, 912 TFLOP/s (600 us with other inputs from
// call to call), the tensor pipe half busy, a pair of tiles about 3700 clocks a key tile; 512 at 0 16
// us, of which 7 are the first scores' way (2500 clocks to set up, Q and the first decode 7000) and the
// output.
// The loops of the five roles have to fit the instruction cache together; where they did not, both SMs
// of a TPC ran a quarter slower at times.
// Every wait is bounded, and a warp's lanes give up together: one that runs out sets the error words,
// and the rows that depend on it (or their parts, and with them the join) come out NaN.
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "kq4.cuh"
#include "kutil.cuh"

namespace gb {

namespace {

constexpr int kRows = 128;        // q rows per tile, tensor-memory lanes
constexpr int kKeys = 128;        // keys per tile
constexpr int kHalf = 64;         // keys whose scores are one product, and one step of the softmax
constexpr int kKWarp0 = 8, kVWarp0 = 12, kMmaWarp = 16;  // groups of 4 warps
constexpr int kThreads = 20 * 32;
// registers per thread: 96 at the launch (640 x 96 = 61440), then split between the warp groups:
// 256 x 120 (softmax) + 256 x 72 (decoding) + 128 x 96 (products) = 61440
constexpr int kSoftRegs = 120, kDecRegs = 72, kMmaRegs = 96;
static_assert(256 * kSoftRegs + 256 * kDecRegs + 128 * kMmaRegs <= kThreads * 96, "register split");
constexpr int kOkRing = 4;        // page masks outlive the K stage they came with
constexpr int kFmaExp = 5;  // see ex2_fma
constexpr float kPShift = 7.0f, kMost = 32768.0f;  // P is exp2(s - m + 7), at most 2^15
constexpr float kLog2e = 1.4426950408889634f;
constexpr long long kSpinCycles = 4000000000LL;  // about 2 s at 1.9 GHz

__device__ int attn_q4_tc_error_word;
std::atomic<bool> expire_waits{false};

template <int HD, bool K2>
struct Tc {
    static constexpr int kTileK = kKeys * HD * 2;  // bytes of a Q, K or V tile
    static constexpr int kSmem = (2 + 2 + 2 + (K2 ? 1 : 0)) * kTileK + 1024;
};

__device__ __forceinline__ uint32_t su32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* b, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(su32(b)), "r"(parity)
        : "memory");
    return done != 0;
}
// bounded wait of a lane; false (and the CTA's abort flag set) when it runs out.  The test itself may
// suspend the warp for the hinted time, so a waiting warp leaves the issue slots to the others
__device__ __forceinline__ bool lane_wait(uint64_t* b, uint32_t parity, volatile int* abort) {
    if (mbar_test(b, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
            " selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(su32(b)), "r"(parity), "r"(10000u)
            : "memory");
        if (done) return true;
        if (*abort) return false;
        if (clock64() - t0 > kSpinCycles) {
            *abort = 1;
            return false;
        }
    }
}
// the same for a warp, whose lanes go on together or give up together: a lane that gave up alone would
// leave the others at their next vote
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort) {
    return __all_sync(0xffffffffu, lane_wait(b, parity, abort));
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* b, bool me) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(
            su32(b)),
        "r"((int)me)
        : "memory");
}
// K-major, 128-byte swizzle: rows of 128 B, 8-row groups 1024 B apart
__device__ __forceinline__ uint64_t desc_sw128(uint32_t a) {
    return (uint64_t)((a & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16, D f32, A and B f16, both K-major, M = 128
constexpr uint32_t idesc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
// Products and commits are issued by the elected lane, as a predicate on the instruction: the whole
// warp runs the same code, so descriptors and addresses stay in uniform registers (an issue every 32
// clocks; under a branch on the lane, or with operands from per-thread registers, about 70 to 115,
// more than the 64 a 128 x 128 x 16 product runs)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add,
                                       bool me) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"((int)add), "r"((int)me)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool add,
                                       bool me) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"((int)add), "r"((int)me)
        : "memory");
}
// 32 columns of the warp's 32 lanes, a lane per thread
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
        "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
        "%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                   "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                   "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
// wait for this thread's loads; the registers are operands, so no use is scheduled before it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                   "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                   "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                   "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                   "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                   "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
        "%14,%15,%16};" ::"r"(t),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
// Loads of the cache.  It does not change after pdl_wait(), so they may move across the barriers (no
// volatile, no memory clobber); but the kernel before may still be writing it when this one starts, so
// they do not take the read-only path of __ldg.  (.cg: 3 to 4% more time, its 16-byte pieces of a row
// come from L2 one by one.)
__device__ __forceinline__ uint32_t ld_u16(const void* p) {
    uint16_t v;
    asm("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_u32(const void* p) {
    uint32_t v;
    asm("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_u32x2(const void* p) {
    uint2 v;
    asm("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 ld_u32x4(const void* p) {
    uint4 v;
    asm("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
        : "l"(p));
    return v;
}
template <int N>
__device__ __forceinline__ void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 2^z of two values on the FMA units: the integer part enters the exponent, the rest, in
// [-1/2, 1/2], a cubic with 2^0 = 1 exact and the least largest relative error, 1.0e-4 (rounding to
// f16 makes 2.4e-4).  -inf gives exactly 0; z above 126, and NaN, something finite above kMost, so
// that the half is done over with the other form.
// One pair of exponentials in kFmaExp takes this way in bf16 calls, whose exponential units (16 a
// clock) are as busy as the products: 2048 tokens at 14336 took 575 us without, 542 with every 5th
// pair, 541 to 567 with every 4th to 16th, 604 with every 2nd (565 with every 5th now; the error of
// such calls against 64 bits is 1.68e-3, of which rounding the output alone makes 1.66e-3).
__device__ __forceinline__ float2 ex2_fma(float2 z) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(z.x));  // -127, 126
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(z.y));
    const float2 big = make_float2(12582912.0f, 12582912.0f);  // 1.5 x 2^23: sums are whole numbers
    const float2 n = add2(z, big), f = sub2(z, sub2(n, big));
    float2 p = fma2(f, make_float2(0.05500892f, 0.05500892f), make_float2(0.24221098f, 0.24221098f));
    p = fma2(p, f, make_float2(0.6932829f, 0.6932829f));
    p = fma2(p, f, make_float2(1.0f, 1.0f));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(n.y) << 23)));
}

// keys that row r of the call sees, r counting (position, head of the group) pairs
__device__ __forceinline__ int row_limit(const AttnQ4Args& a, int64_t pos0, int r) {
    const uint32_t rk = a.Hq / a.c.Hkv;
    return (int)max((int64_t)0, min(pos0 + (uint32_t)r / rk + 1, a.max_kv));
}
// key tiles per CTA when those of a block of rows (the last one sees `keys`) are cut into at most
// `splits` runs
__device__ __forceinline__ int run_tiles(int keys, int splits) {
    const int tiles = (keys + kKeys - 1) / kKeys;
    return max(1, (tiles + splits - 1) / splits);
}
// one run's partial: [HD / 4][row][4] floats (neighbouring rows, threads of the writer, lie together),
// then (m, l) of each row
__host__ __device__ constexpr int64_t part_floats(int block_rows, int64_t hd) {
    return block_rows * (hd + 2);
}

// T: type of q and o; TWO: probabilities in two f16 terms
template <typename T, int HD, bool TWO>
__global__ void __launch_bounds__(kThreads, 1)
    k_attn_q4_tc(const __grid_constant__ AttnQ4Args a, int block_rows, float* parts) {
    pdl_wait();
    // the cache as it is after the wait: no load of it can move before
    const uint8_t *kpool = a.c.k, *vpool = a.c.v;
    const int32_t* pages = a.c.pages;
    asm volatile("" : "+l"(kpool), "+l"(vpool), "+l"(pages));
    constexpr bool K2 = std::is_same<T, __half>::value;  // K in two f16 terms
    using S = Tc<HD, K2>;
    constexpr int NB = HD / 32, VW = HD / 64;
    extern __shared__ __align__(1024) uint8_t raw_smem[];
    uint8_t* smem = raw_smem + ((1024 - (su32(raw_smem) & 1023)) & 1023);
    uint8_t* sQ = smem;                   // [2 tiles]
    uint8_t* sK = sQ + 2 * S::kTileK;     // [2 stages]
    uint8_t* sV = sK + 2 * S::kTileK;
    uint8_t* sL = sV + 2 * S::kTileK;     // K2: second terms, one stage
    __shared__ __align__(8) uint64_t k_full[2][2], k_empty[2][2], v_full[2], v_empty[2], s_full[2][2],
        p_full[2][2], q_full[2], o_most[2], o_full[2], all_done;
    __shared__ __align__(16) uint32_t s_ok[kOkRing][4];
    __shared__ uint32_t s_tmem;
    __shared__ int s_bad[NB];  // per block of V: the first key whose scale was no number
    __shared__ float s_qs[2 * kRows];  // softmax scale of the rows in powers of two
    __shared__ int s_abort;
    volatile int* abort = &s_abort;
    // the warp index and the tensor-memory base come out of a shuffle: uniform to the compiler, so
    // the product warp's operands live in uniform registers
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rk = a.Hq / a.c.Hkv, hk = blockIdx.y;
    // the last rows see the most keys: they start first
    const int rows = (int)a.r.n * rk,  // < 2^30: attn_q4_tc_fits
              row0 = (gridDim.x - 1 - blockIdx.x) * block_rows,
              row1 = min(row0 + block_rows, rows);  // one or two tiles of rows
    const int64_t pos0 = kv_q4_pos(a.r, 0);
    const int64_t slot = kv_q4_slot(a.r, 0);
    auto limit = [&](int r) { return row_limit(a, pos0, r); };
    // this CTA's run of key tiles
    const int block_keys = limit(row1 - 1);
    const int run = run_tiles(block_keys, gridDim.z);
    const int first = __shfl_sync(0xffffffffu, (int)blockIdx.z * run, 0);
    if (first > 0 && first * kKeys >= block_keys) return;
    const bool alone = run * kKeys >= block_keys;  // the only run: it writes the output
    int tiles[2];  // key tiles of each q tile, of this run
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r = min(row0 + (t + 1) * kRows, row1) - 1;
        const int n = r >= row0 + t * kRows ? (limit(r) + kKeys - 1) / kKeys - first : 0;
        // through a shuffle, like the warp index: uniform branches
        tiles[t] = __shfl_sync(0xffffffffu, max(0, min(n, run)), 0);
    }
    const int steps = max(tiles[0], tiles[1]);

    if (tid < NB) s_bad[tid] = INT_MAX;
    if (tid == 0) {
        s_abort = a.expired;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], 1);
            for (int h = 0; h < 2; ++h) {
                mbar_init(&k_full[i][h], 2);
                mbar_init(&k_empty[i][h], 1);
                mbar_init(&s_full[i][h], 1);
                mbar_init(&p_full[i][h], 4);
            }
            mbar_init(&q_full[i], (block_rows == kRows ? 8 : 4) + a.expired);  // (nobody's arrival)
            mbar_init(&o_most[i], 1);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&all_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         su32(&s_tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    auto tS = [&](int i) { return tmem + i * kKeys; };
    auto tO = [&](int i) { return tmem + 2 * kKeys + i * HD; };

    if (warp >= kKWarp0 && warp < kMmaWarp) {
        // ---------------------------------------------------------------- K and V tiles
        regs_down<kDecRegs>();
        const int p = tid & 127;
        const uint32_t page_len = (uint32_t)a.c.page_len;
        const bool in = slot >= 0 && slot < a.c.n_slots;
        const int n = in ? block_keys : 0;
        const int32_t* plist = pages ? pages + slot * a.c.per_slot : nullptr;
        // What is requested ahead: the page id two tiles, the words one tile before they are used;
        // nothing in between looks at a loaded value, so no load is waited for.  A key outside the
        // cache reads the first rows of its pool instead and gets zero scales.
        const int shift = a.shift;
        const uint64_t page_stride = a.c.Hkv * a.c.page_bytes, head = hk * a.c.page_bytes,
                       scales = head + (uint64_t)page_len * (HD / 2);
        auto id_of = [&](int k) {
            if (k >= n) return -1;
            if (!plist) return (int)slot;
            return (int)ld_u32(plist + (shift >= 0 ? (uint32_t)k >> shift : (uint32_t)k / page_len));
        };
        auto rows_at = [&](int k, int pg, bool ok, uint64_t& code, uint64_t& scale) {
            uint32_t prow = k;
            if (plist) prow = shift >= 0 ? (uint32_t)k & (page_len - 1) : (uint32_t)k % page_len;
            if (!ok) prow = 0, pg = 0;
            const uint64_t base = (uint32_t)pg * page_stride;
            code = base + head + (uint64_t)prow * (HD / 2);
            scale = base + scales + (uint64_t)prow * (HD / 16);
        };
        // One copy of the code and one register set: a tile's words are requested when the tile before
        // is decoded, and have until a stage is given back.  The five roles' loops have to fit the
        // instruction cache together: with two sets in turn (this code twice) a seventh of its requests
        // missed, and 2048 tokens at 14336 took 626 us instead of 575.
        auto stream = [&](auto x, auto key, auto fetch, auto decode) {
            int id = id_of(key(0));
            fetch(0, id, x);
            id = id_of(key(1));
#pragma unroll 1
            for (int j = 0; j < steps; ++j) {
                if (!decode(j, x) || j + 1 == steps) break;
                fetch(j + 1, id, x);
                id = id_of(key(j + 2));
            }
        };
        if (warp < kVWarp0) {
            struct Words {  // thread p owns key p of the tile
                uint32_t w[NB * 4], d[NB / 2];
                bool ok;
            };
            stream(
                Words{}, [&](int j) { return (first + j) * kKeys + p; },
                [&](int j, int id, Words& x) {
                    uint64_t code, scale;
                    x.ok = id >= 0 && id < a.c.n_pages;
                    rows_at((first + j) * kKeys + p, id, x.ok, code, scale);
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        const uint4 v = ld_u32x4(kpool + code + 16 * i);
                        x.w[4 * i] = v.x, x.w[4 * i + 1] = v.y;
                        x.w[4 * i + 2] = v.z, x.w[4 * i + 3] = v.w;
                    }
#pragma unroll
                    for (int i = 0; i < NB / 2; ++i)
                        x.d[i] = ld_u32(kpool + scale + 4 * i);
                },
                [&](int j, Words& x) {
                    const int st = j & 1, h = p >> 6;  // stage; half of the tile
                    if (j >= 2 && !mbar_wait(&k_empty[st][h], ((j >> 1) - 1) & 1, abort))
                        return false;
                    uint8_t* dst = sK + st * S::kTileK + p * 128;
                    auto put = [&](uint8_t* to, bool low) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const __half2 d2 = u2h(x.ok ? x.d[b / 2] : 0u);
                            const __half2 d = b & 1 ? __high2half2(d2) : __low2half2(d2);
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                __half2 u[4], k[4];
                                codes(x.w[c * NB + b], u);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    k[i] = __hmul2(u[i], d);
                                    if (low) k[i] = __hfma2(u[i], d, __hneg2(k[i]));
                                }
                                const int ch = (b & 1) * 4 + c;
                                *(uint4*)(to + (b >> 1) * (kKeys * 128) + ((ch ^ (p & 7)) << 4)) =
                                    make_uint4(h2u(k[0]), h2u(k[1]), h2u(k[2]), h2u(k[3]));
                            }
                        }
                    };
                    put(dst, false);
                    if constexpr (K2) {
                        // one stage of second terms: free once the tile before has its scores
                        if (j >= 1 && !mbar_wait(&k_empty[st ^ 1][h], ((j - 1) >> 1) & 1, abort))
                            return false;
                        // decoded anew: keeping the first terms would cost 64 registers
#pragma unroll
                        for (int i = 0; i < NB * 4; ++i) asm volatile("" : "+r"(x.w[i]));
                        put(sL + p * 128, true);
                    }
                    const uint32_t ok = __ballot_sync(0xffffffffu, x.ok);
                    if (lane == 0) s_ok[j % kOkRing][warp - kKWarp0] = ok;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&k_full[st][h]);
                    return true;
                });
        } else {
            // thread: 8 keys 8 kg.. (of one group of 16: one page), words VW vw..
            const int kg = p & 15, vw = p >> 4;
            const int all_see = limit(row0);  // keys below it are seen by every row
            struct Words {
                uint32_t w[8][VW], s[8];
                int keys;  // of the 8 keys, how many are seen
            };
            stream(
                Words{}, [&](int j) { return (first + j) * kKeys + kg * 8; },
                [&](int j, int id, Words& x) {
                    uint64_t code, scale;
                    const int k0 = (first + j) * kKeys + kg * 8;
                    const bool ok = id >= 0 && id < a.c.n_pages;
                    x.keys = ok ? min(8, n - k0) : 0;
                    rows_at(k0, id, ok, code, scale);
                    const uint8_t* src = vpool + code + vw * (VW * 4);
                    const uint16_t* ds = (const uint16_t*)(vpool + scale) + vw * VW / 4;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (VW == 2) {
                            const uint2 v = ld_u32x2(src + i * (HD / 2));
                            x.w[i][0] = v.x, x.w[i][VW - 1] = v.y;
                        } else {
                            x.w[i][0] = ld_u32(src + i * (HD / 2));
                        }
                        x.s[i] = ld_u16(ds + i * NB);
                    }
                },
                [&](int j, Words& x) {
                    const int st = j & 1;
                    if (j >= 2 && !mbar_wait(&v_empty[st], ((j >> 1) - 1) & 1, abort)) return false;
                    uint8_t* dst = sV + st * S::kTileK + (kg >> 3) * (HD * 128);
                    const int k0 = (first + j) * kKeys + kg * 8;
                    if (x.keys < 8 || k0 + 8 > all_see) {
#pragma unroll
                        for (int i = 7; i >= 0; --i) {
                            if (i < x.keys && !bad_scales(x.s[i])) continue;
                            x.s[i] = 0;
                            if (i < x.keys) atomicMin(&s_bad[vw * VW / 4], k0 + i);
                        }
                    }
                    __half2 vd[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vd[i] = u2h(__byte_perm(x.s[2 * i], x.s[2 * i + 1], 0x5410));
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const unsigned sel = hf ? 0x7632u : 0x5410u;
                            __half2 u[4][4];  // [key pair][nibble]
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                codes(__byte_perm(x.w[2 * q][i], x.w[2 * q + 1][i], sel), u[q]);
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                uint4 v;
                                v.x = h2u(__hmul2(u[0][d], vd[0]));
                                v.y = h2u(__hmul2(u[1][d], vd[1]));
                                v.z = h2u(__hmul2(u[2][d], vd[2]));
                                v.w = h2u(__hmul2(u[3][d], vd[3]));
                                const int dim = (vw * VW + i) * 8 + hf * 4 + d;
                                *(uint4*)(dst + dim * 128 + (((kg & 7) ^ (dim & 7)) << 4)) = v;
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[st]);
                    return true;
                });
        }
    } else if (warp >= kMmaWarp) {
        // ---------------------------------------------------------------- products
        regs_down<kMmaRegs>();
        if (warp == kMmaWarp && steps > 0) {
            uint32_t elected;
            asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
                         : "=r"(elected));
            const bool me = elected != 0;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                const bool done = mbar_wait(bar, parity, abort);
                tc_fence_after();
                return done;
            };
            // descriptors of the tiles' starts; a step along K adds 32 bytes (2 in the address field)
            const uint64_t q_at = desc_sw128(su32(sQ)), k_at = desc_sw128(su32(sK)),
                           v_at = desc_sw128(su32(sV)), l_at = desc_sw128(su32(sL));
            constexpr uint64_t kTile = S::kTileK >> 4;
            // scores of keys 64 h .. of tile j; and their share of the output
            auto qk = [&](int i, int j, int h) {
                const uint64_t q = q_at + i * kTile,
                               k = k_at + (j & 1) * kTile + h * (kHalf * 128 >> 4);
                const uint32_t d = tS(i) + h * kHalf;
#pragma unroll
                for (int x = 0; x < HD / 16; ++x) {
                    const uint32_t off = ((x >> 2) * (kRows * 128) + (x & 3) * 32) >> 4;
                    mma_ss(d, q + off, k + off, idesc(kHalf), x > 0, me);
                    if constexpr (K2)
                        mma_ss(d, q + off, l_at + h * (kHalf * 128 >> 4) + off, idesc(kHalf), true, me);
                }
                tc_commit(&s_full[i][h], me);
            };
            auto pv = [&](int i, int j, int h) {
                const uint64_t v = v_at + (j & 1) * kTile + h * (HD * 128 >> 4);
                const uint32_t d = tO(i), p = tS(i) + h * kHalf;
#pragma unroll
                for (int x = 0; x < kHalf / 16; ++x) {
                    const uint64_t b = v + (x * 32 >> 4);
                    // 32 keys: 16 columns of P, then 16 of its second term
                    const uint32_t at = p + (x >> 1) * 32 + (x & 1) * 8;
                    mma_ts(d, at, b, idesc(HD), x > 0 || h > 0 || j > 0, me);
                    if constexpr (TWO) mma_ts(d, at + 16, b, idesc(HD), true, me);
                }
                if (j + 1 == tiles[i]) tc_commit(h ? &o_full[i] : &o_most[i], me);
            };
            bool ok = true;
            for (int i = 0; i < 2; ++i)
                if (ok && tiles[i] > 0) ok = wait(&q_full[i], 0);
            for (int h = 0; h < 2 && ok; ++h) {
                ok = wait(&k_full[0][h], 0);
                if (!ok) break;
                for (int i = 0; i < 2; ++i)
                    if (tiles[i] > 0) qk(i, 0, h);
                tc_commit(&k_empty[0][h], me);
            }
            for (int j = 0; j < steps && ok; ++j) {
                ok = wait(&v_full[j & 1], (j >> 1) & 1);
#pragma unroll 1  // for the instruction cache, too
                for (int h = 0; h < 2; ++h) {
                    bool k_ready = false;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!ok || j >= tiles[i]) continue;
                        ok = wait(&p_full[i][h], j & 1);
                        if (!ok) continue;
                        pv(i, j, h);
                        if (j + 1 < tiles[i]) {
                            if (!k_ready) {
                                ok = wait(&k_full[(j + 1) & 1][h], ((j + 1) >> 1) & 1);
                                if (!ok) continue;
                                k_ready = true;
                            }
                            qk(i, j + 1, h);
                        }
                    }
                    if (ok && j + 1 < steps) tc_commit(&k_empty[(j + 1) & 1][h], me);
                }
                if (ok) tc_commit(&v_empty[j & 1], me);
            }
            // every issued product has completed once this commit arrives
            tc_commit(&all_done, me);
            const long long c0 = clock64();
            bool done = false;
            while (!done && clock64() - c0 < kSpinCycles) done = mbar_test(&all_done, 0);
            if (!done) *abort = 1;
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- softmax, output
        regs_up<kSoftRegs>();
        // Q: a warp loads, scales and stores its 32 rows, HD / 8 lanes a row with 8 dims each; of a
        // block of one tile warps w and w + 4 take 16 rows each (512 tokens at 0: 16.5 -> 15.7 us)
        const bool half = block_rows == kRows;
        const int rows_q = half ? 16 : 32, warp_q = half ? (warp & 3) * 32 + (warp >> 2) * 16 : warp * 32;
        const int t = warp >> 2;
        if (tiles[half ? 0 : t] > 0) {
            constexpr int kLanes = HD / 8, kPer = 32 / kLanes, kFly = sizeof(T) == 4 ? 2 : 4;
            const int w = lane % kLanes;
            const int r0 = warp_q + lane / kLanes;  // the lane's first row, of the block's
            uint32_t i_q = (uint32_t)(row0 + r0) / (uint32_t)rk, h_q = row0 + r0 - i_q * rk;
#pragma unroll 1
            for (int i = 0; i < rows_q; i += kPer * kFly) {
                T x[kFly][8];  // kFly rows are requested before the first is used
#pragma unroll
                for (int f = 0; f < kFly; ++f) {
                    const bool in = row0 + r0 + i + f * kPer < row1;
                    const T* qp = (const T*)a.q + (in ? i_q * a.q_row + (hk * rk + h_q) * a.q_head : 0) +
                                  w * 8;
                    if (a.q_vec) {
                        constexpr int N = 16 / sizeof(T);
#pragma unroll
                        for (int j = 0; j < 8; j += N) *(uint4*)&x[f][j] = *(const uint4*)(qp + j);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[f][j] = qp[j];
                    }
                    if (!in) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) q4_put(&x[f][j], 0.0f);
                    }
                    h_q += kPer;
                    while (h_q >= (uint32_t)rk) h_q -= rk, ++i_q;
                }
#pragma unroll
                for (int f = 0; f < kFly; ++f) {
                    const int r = r0 + i + f * kPer;
                    float y[8], big = 0.0f, bad = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        y[j] = q4_to_f(x[f][j]);
                        big = fmaxf(big, fabsf(y[j]));
                        bad = fmaf(y[j], 0.0f, bad);  // NaN once an element is not finite
                    }
#pragma unroll
                    for (int o = 1; o < kLanes; o <<= 1) {
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                        bad += __shfl_xor_sync(0xffffffffu, bad, o);
                    }
                    // 2^e with big / 2^e in [1, 2); a negative scale moves into q, a zero one
                    // becomes too small to tell scores apart.  A row with an infinity or a NaN is
                    // NaN throughout: NaN scores where it sees a key, and -inf where it does not
                    const int e = min(max((int)(__float_as_uint(big) >> 23) - 127, -126), 126);
                    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                    float down = __uint_as_float((uint32_t)(127 - e) << 23);
                    if (w == 0) s_qs[r] = fmaxf(fabsf(a.scale) * kLog2e * up, 1e-30f);
                    if (a.scale < 0.0f) down = -down;
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = fmaf(y[j], down, bad);
                    uint4 v;
                    v.x = h2u(__floats2half2_rn(y[0], y[4]));
                    v.y = h2u(__floats2half2_rn(y[1], y[5]));
                    v.z = h2u(__floats2half2_rn(y[2], y[6]));
                    v.w = h2u(__floats2half2_rn(y[3], y[7]));
                    const int rt = r & (kRows - 1);
                    *(uint4*)(sQ + (r >> 7) * S::kTileK + rt * 128 + (w >> 3) * (kRows * 128) +
                              (((w & 7) ^ (rt & 7)) << 4)) = v;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();  // s_qs of the warp's rows, too
            if (lane == 0) mbar_arrive(&q_full[half ? 0 : t]);
        }
        const int row = row0 + tid;
        bool ok = true;
        if (half && tiles[t] > 0) ok = mbar_wait(&q_full[t], 0, abort);  // s_qs
        const float qs = tiles[t] > 0 ? s_qs[tid] : 0.0f;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 tensor-memory lanes
        const uint32_t ts = tS(t) + lanes, to = tO(t) + lanes;
        const int lim = row < row1 ? limit(row) : 0;
        // keys below this are seen by every row of the warp
        const int wr = row0 + warp * 32;
        const int full = wr + 31 < row1 ? limit(wr) : 0;
        // a row without keys in this run needs no maximum
        float m = lim > first * kKeys ? -INFINITY : 0.0f, l = 0.0f;
        uint32_t va[32], vb[32];
        // halves of the key tiles in turn: while one is worked on here, the products of the other run
        for (int step = 0; step < 2 * tiles[t] && ok; ++step) {
            const int j = step >> 1, h = step & 1;
            ok = mbar_wait(&s_full[t][h], j & 1, abort);
            if (!ok) break;
            tc_fence_after();
            const uint32_t tp = ts + h * kHalf;
            const int k0 = (first + j) * kKeys + h * kHalf;
            const uint2 pages = *(const uint2*)(s_ok[j % kOkRing] + 2 * h);
            const bool all = k0 + kHalf <= full && (pages.x & pages.y) == 0xffffffffu;
            // key i of the 32 at k0 + 32 c is not seen: -inf
            auto mask = [&](uint32_t (&v)[32], int c) {
                const int left = max(0, min(32, lim - k0 - c * 32));
                const uint32_t seen = (c ? pages.y : pages.x) & (uint32_t)((1ull << left) - 1);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (!(seen & (1u << i))) v[i] = 0xFF800000u;
            };
            auto load = [&] {
                tmem_ld32(tp, va);
                tmem_ld32(tp + 32, vb);
                tmem_wait_ld(va);
                tmem_wait_ld(vb);
                if (!all) {
                    mask(va, 0);
                    mask(vb, 1);
                }
            };
            // The largest score of these columns renews the maximum; O and l are scaled.  O must be
            // still: the product before it has completed once the other half's next scores (or, past
            // the last tile, o_most) are there, and the next one waits for this P.
            auto renew = [&] {
                float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    y[i & 2] = fmaxf(fmaxf(y[i & 2], __uint_as_float(va[i])),
                                     __uint_as_float(va[i + 1]));
                    y[(i & 2) + 1] = fmaxf(fmaxf(y[(i & 2) + 1], __uint_as_float(vb[i])),
                                           __uint_as_float(vb[i + 1]));
                }
                const float x = fmaxf(m, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) * qs);
                const float f = ex2(m - (x == -INFINITY ? 0.0f : x));
                m = x;
                l *= f;
                if (step == 0) return true;
                uint64_t* still = h == 0            ? &s_full[t][1]
                                  : j + 1 < tiles[t] ? &s_full[t][0]
                                                     : &o_most[t];
                const uint32_t parity = h == 0 ? j & 1 : j + 1 < tiles[t] ? (j + 1) & 1 : 0;
                if (!mbar_wait(still, parity, abort)) return false;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                    uint32_t u[16];
                    tmem_ld16(to + c * 16, u);
                    tmem_wait_ld(u);
#pragma unroll
                    for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * f);
                    tmem_st16(to + c * 16, u);
                }
                return true;
            };
            float2 sum[2];
            // P in the registers of the scores
            auto probs = [&](uint32_t (&v)[32], float2& total, auto exact) {
                const float ref = kPShift - (m == -INFINITY ? 0.0f : m);
                const float2 qs2 = make_float2(qs, qs), ref2 = make_float2(ref, ref);
                float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 z = fma2(make_float2(__uint_as_float(v[2 * i]),
                                                      __uint_as_float(v[2 * i + 1])), qs2, ref2);
                    const float2 p = !decltype(exact)::value && !TWO && i % kFmaExp == 0
                                         ? ex2_fma(z)
                                         : make_float2(ex2(z.x), ex2(z.y));
                    part[i & 1] = add2(part[i & 1], p);
                    v[2 * i] = __float_as_uint(p.x);
                    v[2 * i + 1] = __float_as_uint(p.y);
                }
                total = add2(part[0], part[1]);
            };
            auto store = [&](const uint32_t (&v)[32], int c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 p =
                        make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                    const __half2 q = __floats2half2_rn(p.x, p.y);
                    hi[i] = h2u(q);
                    if constexpr (TWO) {
                        const float2 f = __half22float2(q);
                        lo[i] = h2u(__floats2half2_rn(p.x - f.x, p.y - f.y));
                    }
                }
                tmem_st16(tp + c * 32, hi);
                if constexpr (TWO) tmem_st16(tp + c * 32 + 16, lo);
            };
            load();
            if (__any_sync(0xffffffffu, m == -INFINITY)) ok = renew();  // the first half, as a rule
            probs(va, sum[0], std::false_type{});
            probs(vb, sum[1], std::false_type{});
            sum[0] = add2(sum[0], sum[1]);
            // a P too large for f16 shows in the sum (they are positive): once more, with the maximum
            if (__any_sync(0xffffffffu, sum[0].x + sum[0].y > kMost)) {
                load();
                ok &= renew();
                probs(va, sum[0], std::true_type{});
                probs(vb, sum[1], std::true_type{});
                sum[0] = add2(sum[0], sum[1]);
            }
            l += sum[0].x + sum[0].y;
            store(va, 0);
            store(vb, 1);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t][h]);
        }
        // not earlier: CTAs of the next launch would take the SMs that a small grid leaves free, and then
        // share TPCs (measured at 333 tokens at 1999: 76 us instead of 73)
        pdl_launch();
        if (ok && tiles[t] > 0) {
            ok = mbar_wait(&o_full[t], 0, abort);
            tc_fence_after();
        }
        {
            float r = alone ? (l != 0.0f ? 1.0f / l : 0.0f) : 1.0f;
            if (l == 0.0f) m = -INFINITY;  // (of a row without keys in this run)
            if (!ok) r = m = l = __int_as_float(0x7FFFFFFF);
            const uint32_t i_o = (uint32_t)row / (uint32_t)rk, h_o = row - i_o * rk;
            T* op = (T*)a.o + ((int64_t)i_o * a.Hq + hk * rk + h_o) * HD;
            float* part = parts + (((int64_t)(gridDim.x - 1 - blockIdx.x) * a.c.Hkv + hk) * gridDim.z +
                                   blockIdx.z) * part_floats(block_rows, HD);
#pragma unroll 1  // for the instruction cache, like the masks' few instructions
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t v[32];
                if (tiles[t] > 0 && ok) {
                    tmem_ld32(to + c * 32, v);
                    tmem_wait_ld(v);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0;
                }
                if (lim > s_bad[c]) {  // (V's warps are done: their last stage has been multiplied)
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0x7FFFFFFFu;
                }
                if (row < row1 && alone) {
                    constexpr int N = 16 / sizeof(T);
#pragma unroll
                    for (int i = 0; i < 32; i += N) {
                        uint4 raw;
                        T* e = (T*)&raw;
#pragma unroll
                        for (int k = 0; k < N; ++k) q4_put(e + k, __uint_as_float(v[i + k]) * r);
                        *(uint4*)(op + c * 32 + i) = raw;
                    }
                } else if (row < row1) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *(uint4*)(part + ((c * 8 + i / 4) * block_rows + tid) * 4) =
                            make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            if (row < row1 && !alone)
                *(float2*)(part + block_rows * HD + tid * 2) = make_float2(m, l);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        if (*abort) {
            attn_q4_tc_error_word = 1;
            if (a.err) *(volatile int*)a.err = 1;  // mapped host memory
        }
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// Joins the runs of 8 rows per CTA, thread (row, groups of 4 dims); rows of a block that ran alone are
// written already.
template <typename T, int HD>
__global__ void __launch_bounds__(128)
    k_attn_q4_tc_join(const __grid_constant__ AttnQ4Args a, int block_rows, int splits,
                      const float* parts) {
    pdl_launch();
    pdl_wait();
    const int rk = a.Hq / a.c.Hkv, hk = blockIdx.y, rows = (int)a.r.n * rk;
    const int row0 = blockIdx.x * 8, block = row0 / block_rows;  // blocks are multiples of 8 rows
    const int keys = row_limit(a, kv_q4_pos(a.r, 0), min((block + 1) * block_rows, rows) - 1);
    const int run = run_tiles(keys, splits);
    const int n = (keys + run * kKeys - 1) / (run * kKeys);  // runs
    const int row = row0 + threadIdx.x % 8, r = row - block * block_rows, g = threadIdx.x / 8;
    if (n <= 1 || row >= rows) return;
    const int64_t pf = part_floats(block_rows, HD);
    const float* p = parts + ((int64_t)block * a.c.Hkv + hk) * splits * pf;
    constexpr int N = HD / 64;  // groups of 4 dims per thread: g, g + 16
    float m = -INFINITY, l = 0.0f;
    float4 acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
        const float* q = p + i * pf;
        const float2 ml = __ldcg((const float2*)(q + block_rows * HD + r * 2));
        float4 v[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            v[k] = __ldcg((const float4*)(q + ((k * 16 + g) * block_rows + r) * 4));
        const float x = fmaxf(m, ml.x), ref = x == -INFINITY ? 0.0f : x;
        const float old = ex2(m - ref), now = ex2(ml.x - ref);
        m = x;
        l = fmaf(l, old, ml.y * now);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            acc[k].x = fmaf(acc[k].x, old, v[k].x * now), acc[k].y = fmaf(acc[k].y, old, v[k].y * now);
            acc[k].z = fmaf(acc[k].z, old, v[k].z * now), acc[k].w = fmaf(acc[k].w, old, v[k].w * now);
        }
    }
    const float f = l != 0.0f ? 1.0f / l : 0.0f;
    const uint32_t i_o = (uint32_t)row / (uint32_t)rk, h_o = row - i_o * rk;
    T* o = (T*)a.o + ((int64_t)i_o * a.Hq + hk * rk + h_o) * HD;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        T* d = o + (k * 16 + g) * 4;
        q4_put(d, acc[k].x * f), q4_put(d + 1, acc[k].y * f);
        q4_put(d + 2, acc[k].z * f), q4_put(d + 3, acc[k].w * f);
    }
}

// The cut of a launch: rows per CTA (one or two tiles) and runs of key tiles per row block, by the
// time it takes, in us: CTAs run one per SM in waves; a CTA costs its key tiles (kTwo with two row
// tiles, kOne with one, whose decode of K and V then serves half the rows) and kFixed besides (Q, the
// first decode, the output), the join of several runs kJoin.  The number of partials is bounded.  The
// constants are those of a first measurement; nearer ones (2.1, 1.35, 8 or 6 in bf16; 3.0 to 3.7 for a
// pair of tiles in f16) chose no better over 54 shapes of 200..1000 tokens at 0..3000 (0 to 0.7% longer).
constexpr double kTwo = 2.4, kOne = 1.5, kFixed = 9.0, kJoin = 5.0;
struct TcPlan {
    int block_rows, splits;
    int64_t blocks;
    double us;
};
TcPlan tc_plan(int64_t n_rows, int64_t rk, int64_t Hkv, int64_t keys, int sms) {
    TcPlan p{};
    const int64_t tiles = std::max<int64_t>(1, (keys + kKeys - 1) / kKeys);
    for (int two = 1; two >= 0; --two) {
        const int block_rows = two ? 2 * kRows : kRows;
        const int64_t blocks = (n_rows * rk + block_rows - 1) / block_rows, base = blocks * Hkv;
        for (int64_t s = 1; s <= tiles && (s == 1 || base * s <= 2 * sms); ++s) {
            const int64_t waves = (base * s + sms - 1) / sms, run = (tiles + s - 1) / s;
            const double us = waves * (run * (two ? kTwo : kOne) + kFixed) + (s > 1 ? kJoin : 0.0);
            if (p.blocks == 0 || us < p.us) p = {block_rows, (int)s, blocks, us};
        }
    }
    return p;
}
int64_t keys_of(const AttnQ4Args& a) {  // what the last row sees, as far as the host knows
    if (a.r.step_pos) return a.max_kv;
    return std::max<int64_t>(0, std::min(a.r.pos0 + a.r.n, a.max_kv));
}
int current_sms() {
    int dev = 0;
    GB_CUDA(cudaGetDevice(&dev));
    return sm_count(dev);
}

template <typename T, int HD, bool TWO>
void launch_tc(const AttnQ4Args& a, cudaStream_t st) {
    using S = Tc<HD, std::is_same<T, __half>::value>;
    int dev = 0;
    GB_CUDA(cudaGetDevice(&dev));
    static std::atomic<bool> ready[64];
    if (dev >= 64 || !ready[dev]) {
        GB_CUDA(cudaFuncSetAttribute(k_attn_q4_tc<T, HD, TWO>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        if (dev < 64) ready[dev] = true;
    }
    const int rk = a.Hq / a.c.Hkv;
    const TcPlan plan = tc_plan(a.r.n, rk, a.c.Hkv, keys_of(a), sm_count(dev));
    GB_CHECK(a.c.Hkv <= 65535, "attn_q4: too many heads for one launch");
    AttnQ4Args b = a;
    b.shift = kv_q4_shift(a.c);
    b.q_vec = kv_q4_vectors(a);
    b.expired = expire_waits;
    float* parts = (float*)((char*)a.work + attn_q4_parts_offset());
    launch_pdl(k_attn_q4_tc<T, HD, TWO>, dim3((unsigned)plan.blocks, a.c.Hkv, plan.splits),
               dim3(kThreads), S::kSmem, st, b, plan.block_rows, parts);
    GB_CUDA(cudaGetLastError());
    if (plan.splits > 1)
        launch_pdl(k_attn_q4_tc_join<T, HD>, dim3((unsigned)((a.r.n * rk + 7) / 8), a.c.Hkv),
                   dim3(128), 0, st, b, plan.block_rows, plan.splits, (const float*)parts);
}

template <typename T, bool TWO>
void launch_tc_hd(const AttnQ4Args& a, cudaStream_t st) {
    if (a.c.hd == 64)
        launch_tc<T, 64, TWO>(a, st);
    else
        launch_tc<T, 128, TWO>(a, st);
}

}  // namespace

bool tc_head_dim(int64_t hd) { return hd == 64 || hd == 128; }

// bytes of the partials behind attn_q4_parts_offset(): at most two CTAs an SM leave one
size_t attn_q4_tc_parts(int64_t hd) {
    return tc_head_dim(hd) ? (size_t)(2 * current_sms() * part_floats(2 * kRows, hd) * 4) : 0;
}

double attn_q4_tc_us(const AttnQ4Args& a) {
    return tc_plan(a.r.n, a.Hq / a.c.Hkv, a.c.Hkv, keys_of(a), current_sms()).us;
}

bool attn_q4_tc_fits(const AttnQ4Args& a) {
    return !a.r.pos && !a.r.slot && tc_head_dim(a.c.hd) &&
           a.r.n * (a.Hq / a.c.Hkv) < (int64_t(1) << 30) &&
           (a.type == kTypeF16 || a.type == kTypeBF16 || (a.type == kTypeF32 && a.fast_f32)) &&
           ((uintptr_t)a.o & 15) == 0;
}

void launch_attn_q4_tc(const AttnQ4Args& a, cudaStream_t st) {
    if (a.type == kTypeF32)
        launch_tc_hd<float, true>(a, st);
    else if (a.type == kTypeF16)
        launch_tc_hd<__half, true>(a, st);
    else
        launch_tc_hd<__nv_bfloat16, false>(a, st);
    GB_CUDA(cudaGetLastError());
}

void attn_q4_tc_expire_waits(bool on) { expire_waits = on; }

void attn_q4_tc_clear_error() {
    const int v = 0;
    GB_CUDA(cudaMemcpyToSymbol(attn_q4_tc_error_word, &v, sizeof v));
}

int attn_q4_tc_error() {
    int v = 0;
    GB_CUDA(cudaMemcpyFromSymbol(&v, attn_q4_tc_error_word, sizeof v));
    return v;
}

}  // namespace gb
