// Packed prompts over the 4-bit cache on the 5th-generation tensor cores.
//
// A block takes 128 query rows of one key/value head: 128 / R consecutive tokens of one sequence times the R query heads that share the head, so that a
// key or value is brought and converted once for all of them.  It walks the cached rows in tiles of 64:
//   S = Q·Kᵀ    Q in fp16 halves hi + lo of the rotated row times a power of two (22 bits); a stored key, code · scale, is exact in fp16: two MMAs
//   P = 2^(S·c − m + 9) per row, in halves hi + lo again, written over S in tensor memory, from where it is the A operand of
//   O += P·V    with O in tensor memory as well
//   warps 0-3   a thread is a row: running maximum and sum of the softmax in fp32, no exchange between lanes.  O is multiplied by the change of the
//               maximum only when a weight would leave fp16 (see kLift)
//   warps 4-11  four for keys, four for values, sixteen rows of a tile each: bulk copies into a place of their own, the codes into registers, and when the
//               tile is free 4-bit codes → fp16 with 128-byte swizzle
//   warp 12     issues the MMAs: Q·K of the next tile before P·V of this one
// The chain from scores over weights to values leaves every unit idle most of the time, and a satisfied wait on a barrier costs 170 cycles: two blocks
// share an SM (half of its tensor and shared memory each: two S/P buffers of 64 columns, O, one tile of keys and one of values).  One block per SM with
// tiles of 128 keys and two of each took 3900 cycles for 128 keys, where the MMAs take 2048.
// Where tiles of queries are few, up to four blocks (a cluster) share the keys of one and join their outputs through shared memory, a part of the rows each.
// Measured: 2048 tokens of 32 heads of 128 86 µs (800 TFLOP/s counting the halves; 101 µs with cold caches), 6000 of 32/8 heads 510 µs (1150).  Bound by the chain
// of a tile (2900 cycles with two blocks on an SM) and by what a block does before its first and after its last tile (25000 cycles).
// Every wait is bounded (codes 341-350 in the device error word).
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "q4_cache.cuh"
#include "tc_common.cuh"
#include <cuda_fp16.h>

namespace dj {
namespace {

constexpr int kPT = 128;                          // query rows of a tile
constexpr int kKT = 64;                           // keys of a tile: two pages
constexpr int kPThreads = 416;                    // warps: 4 softmax, 8 conversion, MMAs

struct PrefillParams {
    const float* qkv; int q_off, ld;
    const unsigned char* cache; int maxSeq, pages;
    const float* starts; const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    float* out; int ldo; int B, H, G, ratio, M; float scale;            // scale: 1/sqrt(hd) · log2(e)
    float* stats; int window;                     // [M][H][2] base (log2) and sum of the weights to it of the last `window` tokens' rows, or null
    const float* acc; float* accOut;
    int* error;
    float* totals;                                // [block][128][hd] for the blocks of clusters
    int splits, least;                            // blocks (a cluster) that share the keys of a tile of queries, tiles of keys to one at least
};
constexpr int kMaxSplits = 4;
// Tiles whose values are summed in tensor memory.  Those sums are cut off, not rounded: values of one sign lose 5.6e-9 of their sum a key, 3.4e-5 at 6000 keys.
// So a sum of 16 tiles goes to memory, where it is added rounded: 5e-6 from 4000 to 65000 keys (32 tiles: 1.1e-5), for 3 % of the time at 1500 keys and 6 % at
// 6000.  For values of both signs, 6000 tokens of 32/8 heads: 1.8e-6, with 10 tiles 1.3e-6 and 5 % more time, with 8 1.2e-6 and 8 %, plain fp32 0.8e-6.
// The sums of the weights go the same way, a tile's and then sixteen tiles' by themselves: a chain of 16 thousand equal weights was off by 1e-4.
constexpr int kSegment = 16;
// A row's weights are taken to a base 2^9 below its maximum, P up to 2^9, and the base stays until one would be above 2^15, the last power of two in fp16.  Steps of
// fp16 end at 2^-24: with the maximum at 2^9, a weight is off by at most 2^-33 of the row's largest (two halves, half a step each).  With the maximum at 1, weights under
// 2^-14 of it kept 10 bits and fewer, those under 2^-25 none: thousands of keys 10 … 18 nats below one were off by up to all of their sum.
constexpr float kLift = 9.0f, kTop = 15.0f;
// The base for a maximum; from 2^27 on a step of a score is more than the lift.
__device__ __forceinline__ float base_of(float most) { return most - (most - kLift) > kTop ? most : most - kLift; }

constexpr size_t kAlone = 120 * 1024;             // more than half of an SM's shared memory
template <int NB> struct PrefillShape {
    static constexpr int HD = 32 * NB, kChunks = (HD + 63) / 64;         // 128-byte pieces of a row
    static constexpr int kQ = kChunks * kPT * 128, kKV = kChunks * kKT * 128;      // bytes of a tile of queries (hi or lo), of keys or values
    static constexpr int kKAt = 2 * kQ, kVAt = kKAt + kKV, kRawAt = kVAt + kKV, kRaw = 16 * (Q4Page<NB>::kRow + 2 * NB);      // kRaw: sixteen rows' codes and scales
    static constexpr size_t kUsed = (size_t)kRawAt + 8 * kRaw + 1024;
    static constexpr size_t kSmem = kUsed > 80 * 1024 ? kUsed : 80 * 1024;         // two blocks per SM: they hold all tensor memory
};

// K-major, 128-byte swizzle: 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3fff) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// MN-major: 64 dims to a 128-byte row, 8-key groups 1024 bytes apart, the next 64 dims kKT rows on
__device__ __forceinline__ uint64_t desc_mn(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3fff) | ((uint64_t)(kKT * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// a, b → packed fp16 and packed remainders
__device__ __forceinline__ void split_half(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = half2_bits(a - f.x, b - f.y);
}
template <int NB> __device__ __forceinline__ void piece_of(uint32_t (&w)[NB], const unsigned char* p) {
    if constexpr (NB == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if constexpr (NB == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

// A tile's row has its dims in the order in which a page word gives them: 16 bytes are word (t, j), its values dims 32j + 4t + {0, 2, 16, 18, 1, 3, 17, 19}.
// Queries are laid down in the same order; outputs are put back when they are stored.
// Bits 6 … 9 of a half of 16 + u are u, the code + 8: (word moved & 0x03c0) ^ 0x4e00 = 24 + code, and (24 + code)·scale - 24·scale = code · scale in one
// fused operation.  24·scale has 10 bits; where it would leave fp16 (scales above 2729) the code is formed first.
__device__ __forceinline__ uint32_t half_of(uint32_t moved, __half2 scale, __half2 off, bool wide) {
    const uint32_t x = (moved & 0x03c003c0u) ^ 0x4e004e00u;
    const __half2 v = *reinterpret_cast<const __half2*>(&x);
    const __half2 r = wide ? __hmul2(__hsub2(v, __float2half2_rn(24.0f)), scale) : __hfma2(v, scale, off);
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <int NB, int ROWS, bool WIDE>
__device__ __forceinline__ void convert_words(const unsigned char* half, int lane, unsigned char* tile, int row, const __half2 (&scale)[NB], int t0, int t1) {
    __half2 off[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) off[j] = __hmul2(scale[j], __float2half2_rn(-24.0f));
#pragma unroll 1
    for (int t = t0; t < t1; t++) {               // rolled: the roles of a block run side by side and share the instruction cache
        uint32_t w[NB];
        piece_of<NB>(w, half + Q4Page<NB>::word(lane, t, 0));
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int c = 4 * j + t;
            *reinterpret_cast<uint4*>(tile + (j >> 1) * (ROWS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                make_uint4(half_of(w[j] << 6, scale[j], off[j], WIDE), half_of(w[j] << 2, scale[j], off[j], WIDE), half_of(w[j] >> 2, scale[j], off[j], WIDE),
                           half_of(w[j] >> 6, scale[j], off[j], WIDE));
        }
    }
}
// Pieces t0, t0 + 1 of a row, in registers, → row `row` of an fp16 tile of ROWS rows.
template <int NB, int ROWS>
__device__ __forceinline__ void convert_pieces(const uint32_t (&w)[2][NB], const float (&s)[NB], unsigned char* tile, int row, int t0) {
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < NB; j++) most = fmaxf(most, s[j]);
    auto all = [&](bool wide) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const __half2 scale = __float2half2_rn(s[j]), off = __hmul2(scale, __float2half2_rn(-24.0f));
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int c = 4 * j + t0 + u;
                *reinterpret_cast<uint4*>(tile + (j >> 1) * (ROWS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                    make_uint4(half_of(w[u][j] << 6, scale, off, wide), half_of(w[u][j] << 2, scale, off, wide), half_of(w[u][j] >> 2, scale, off, wide),
                               half_of(w[u][j] >> 6, scale, off, wide));
            }
        }
    };
    if (__any_sync(0xffffffffu, most > 2048.0f)) all(true); else all(false);
}
// Row `lane` of a page's K or V half, its words (t0 … t1 - 1, j) → row `row` of an fp16 tile of ROWS rows.
template <int NB, int ROWS>
__device__ __forceinline__ void convert_row(const unsigned char* half, int lane, unsigned char* tile, int row, int t0, int t1) {
    __half2 scale[NB];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        const float s = __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(half + Q4Page<NB>::kKs + (lane * NB + j) * 2) << 16);
        most = fmaxf(most, s);
        scale[j] = __float2half2_rn(s);
    }
    if (__any_sync(0xffffffffu, most > 2048.0f)) convert_words<NB, ROWS, true>(half, lane, tile, row, scale, t0, t1);
    else convert_words<NB, ROWS, false>(half, lane, tile, row, scale, t0, t1);
}
template <int NB, int ROWS>
__device__ __forceinline__ void zero_row(unsigned char* tile, int row, int t0, int t1) {
#pragma unroll 1
    for (int c = 0; c < 4 * NB; c++)
        if ((c & 3) >= t0 && (c & 3) < t1) *reinterpret_cast<uint4*>(tile + (c >> 3) * (ROWS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
}

// Query rows of a tile, rotated, in halves of fp16 times a power of two → tiles hi and lo, a row to 4·NB lanes of eight values each, one 16-byte piece;
// `place(row, m, head, position)` says which one row `row` of the first `rows` is, and whether it is one (false: zeros, but the place can be read).
// factors[row] makes a sum of products a score in log2 units (NaN where the row holds an infinity or a NaN).  It is a power of two, 1/sqrt(hd) · log2(e) goes
// into the values: a score is then exact, and the one that its row's base was taken from comes to the lift again, however large scores are.
// Four values to a lane took 12000 cycles a tile of four heads a token, eight 9000.  Loads of several rows ahead cost more in code than they give: the roles
// of a block share the instruction cache (eight prompts of 1500: 303 µs as it is, 307 and 319 with two and three rows ahead).
template <int NB, typename Place>
__device__ __forceinline__ void query_rows(const PrefillParams& p, int warp, int warps, int lane, unsigned char* hi, unsigned char* lo, float* factors, int rows, Place place) {
    constexpr int HD = 32 * NB, LPR = 4 * NB, RPW = 32 / LPR;
    const int c = lane % LPR, dim = (c >> 2) * 32 + (c & 3) * 4;         // this lane's piece, word (c % 4, c / 4): its dims dim … dim + 3, and 16 on
    const float* const q0 = p.qkv + p.q_off + dim;
    const int at = (c >> 3) * (kPT * 128);
#pragma unroll 1
    for (int r = warp * RPW + lane / LPR; r < rows; r += warps * RPW) {
        int m, head, position;
        const bool on = place(r, m, head, position);
        const float* const from = q0 + (size_t)m * p.ld + head * HD;
        const size_t tab = (size_t)position * (HD / 2) + (dim >> 1);
        float4 y[2];
        float2 cs[2], sn[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            y[h] = __ldcg(reinterpret_cast<const float4*>(from + 16 * h));
            cs[h] = *reinterpret_cast<const float2*>(p.cosT + tab + 8 * h);      // the heads of a token share them: through L1
            sn[h] = *reinterpret_cast<const float2*>(p.sinT + tab + 8 * h);
        }
        float most = 0.0f, none = 0.0f;           // none: NaN where a value is an infinity or a NaN
#pragma unroll
        for (int h = 0; h < 2; h++) {
            y[h] = q4_rotate(y[h], cs[h], sn[h]);
            y[h] = make_float4(y[h].x * p.scale, y[h].y * p.scale, y[h].z * p.scale, y[h].w * p.scale);
            most = fmaxf(most, q4_most(y[h]));
            none = fmaf(y[h].x, 0.0f, fmaf(y[h].y, 0.0f, fmaf(y[h].z, 0.0f, fmaf(y[h].w, 0.0f, none))));
        }
        if (none != none) most = INFINITY;
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // the largest value comes to 256 … 512
        most = fmaxf(most, 7.8886091e-31f);
        const int bits = __float_as_int(most) & 0x7f800000;
        const bool fine = most < INFINITY;
        const float mul = __uint_as_float((262u << 23) - (uint32_t)bits);        // 2^(8 - exponent): a normal number for every finite row
        uint4 h = make_uint4(0, 0, 0, 0), l = h;
        if (fine && on) {
            split_half(y[0].x * mul, y[0].z * mul, h.x, l.x);
            split_half(y[1].x * mul, y[1].z * mul, h.y, l.y);
            split_half(y[0].y * mul, y[0].w * mul, h.z, l.z);
            split_half(y[1].y * mul, y[1].w * mul, h.w, l.w);
        }
        const int to = at + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(hi + to) = h;
        *reinterpret_cast<uint4*>(lo + to) = l;
        if (c == 0) factors[r] = fine || !on ? __int_as_float(bits) * (1.0f / 256.0f) : __int_as_float(0x7fc00000);
    }
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)), "l"(reinterpret_cast<const unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// what a block that gives up still has on its way
__device__ __forceinline__ void wait_out(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < 1 << 16 && !mbar_try_wait(bar, parity); i++) {}
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// what block `rank` of the cluster holds at this block's address
__device__ __forceinline__ uint32_t peer_address(uint32_t at, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    return a;
}
__device__ __forceinline__ float2 peer_float2(uint32_t at, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer_address(at, rank)));
    return v;
}
__device__ __forceinline__ float4 peer_float4(uint32_t at, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_address(at, rank)));
    return v;
}

// Sequence, its place and the first token of query tile `tile`, the last tile of a sequence first; whole warps call it.
__device__ __forceinline__ bool tile_of(const PrefillParams& p, int tile, int tokensPerTile, int lane, int& b, int& first, int& tokens, int& t0, int& len, int& pos) {
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        int from = 0, n = 0, l = 0, q = 0;
        if (b0 + lane < p.B) {
            n = q4_rows(__ldcg(p.starts + b0 + lane), __ldcg(p.starts + b0 + lane + 1), p.M, from);
            l = q4_int(__ldcg(p.len + b0 + lane)); q = q4_int(__ldcg(p.pos + b0 + lane));
        }
        const int tiles = (n + tokensPerTile - 1) / tokensPerTile;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < upto);
        if (hit) {
            const int k = __ffs(hit) - 1;
            b = b0 + k;
            first = __shfl_sync(0xffffffffu, from, k);
            tokens = __shfl_sync(0xffffffffu, n, k);
            len = __shfl_sync(0xffffffffu, l, k); pos = __shfl_sync(0xffffffffu, q, k);
            t0 = (__shfl_sync(0xffffffffu, upto, k) - 1 - tile) * tokensPerTile;
            return true;
        }
        tile -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <int NB>
__global__ void __launch_bounds__(kPThreads, 2) k_q4_prefill(const PrefillParams p) {
    using S = PrefillShape<NB>;
    constexpr int HD = S::HD;
    constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kKT >> 3) << 17) | ((uint32_t)(kPT >> 4) << 24);      // fp16 × fp16 → fp32
    constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kPT >> 4) << 24);      // B MN-major
    constexpr uint32_t kO = 2 * kKT;              // O's first column
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bar[8 + 10];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ float s_factor[kPT];
    // what the loops need seldom or only behind them, so that it takes no registers
    __shared__ float* s_out[kPT];                 // a row's place in the output; null: no row of a token
    __shared__ int s_stat[kPT];                   // and in the statistics, or -1
    __shared__ float s_since[kPT];                // what a row's total has to be multiplied by
    __shared__ float s_weights[kPT];              // a row's total of weights
    __shared__ float2 s_row[kPT];                 // a row's base and sum, for the other blocks of the cluster
    __shared__ volatile int s_parts, s_rows;
    __shared__ int4 s_place[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
    constexpr int PITCH = HD + 4, LPR = 8 * NB, RPW = 32 / LPR;         // rows on their way out: floats of one, lanes of one, rows of a warp
    const uint32_t kFull = bar(8), kEmpty = bar(9), vFull = bar(10), vEmpty = bar(11);      // one phase a tile; bars 0-7: the conversion warps' copies
    auto sFull = [&](int s) { return bar(12 + s); };
    auto pReady = [&](int s) { return bar(14 + s); };
    // done: the last product.  Its phase of vEmpty cannot be waited for by those that may not have seen the one before: parities name two phases.
    const uint32_t qReady = bar(16), done = bar(17);
    if (tid == 0) {
        for (int s = 0; s < 8; s++) mbar_init(bar(s), 1);
        mbar_init(kFull, 4); mbar_init(kEmpty, 1); mbar_init(vFull, 4); mbar_init(vEmpty, 1);
        for (int s = 0; s < 2; s++) { mbar_init(sFull(s), 1); mbar_init(pReady(s), 4); }
        mbar_init(qReady, 12);
        mbar_init(done, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tmem_alloc(smem_u32(&s_tmem), 256);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // The kernel before is the append, which has passed its own wait: all but the rows that it writes is complete, so the queries are laid down before it ends.
    const int work = blockIdx.x / p.splits, rank = blockIdx.x - work * p.splits, g = work % p.G, tokensPerTile = kPT / p.ratio;
    if (warp == 12) {                             // one warp looks for the tile's place
        int b = 0, first = 0, tokens = 0, t0 = 0, len = 0, pos = 0, room = 0;
        if (tile_of(p, work / p.G, tokensPerTile, lane, b, first, tokens, t0, len, pos)) room = q4_room(tokens, len, p.maxSeq, pos, p.maxPos);
        if (lane == 0) { s_place[0] = make_int4(b, first + t0, t0, room); s_place[1] = make_int4(len + t0, pos + t0, 0, 0); }
    }
    __syncthreads();
    const int b = s_place[0].x, firstToken = s_place[0].y, t0 = s_place[0].z, room = s_place[0].w, len0 = s_place[1].x, pos0 = s_place[1].y;      // of the tile's first token
    const int used = max(0, min(tokensPerTile, room - t0));              // tokens of this tile
    const int keys = used > 0 ? len0 + used : 0, allTiles = (keys + kKT - 1) / kKT;
    // this block's share: tiles from skip on, its keys, pages and tiles count from there
    const int parts = p.splits > 1 ? min(p.splits, max(1, allTiles / p.least)) : 1;
    const int skip = rank < parts ? allTiles * rank / parts : 0, tiles = rank < parts ? allTiles * (rank + 1) / parts - skip : 0;
    const int pages = (keys + kQ4Page - 1) / kQ4Page - 2 * skip;

    const int inverse = 65535 / p.ratio + 1;      // r · inverse / 2^16 is r / ratio for a row r of the tile
    auto queries = [&]() {                        // twelve warps lay the queries down
        query_rows<NB>(p, warp, 12, lane, smem, smem + S::kQ, s_factor, kPT, [&](int r, int& qm, int& qh, int& qp) {
            const int t = min(r * inverse >> 16, used - 1);
            qm = firstToken + t; qh = g * p.ratio + min(r - t * p.ratio, p.ratio - 1); qp = pos0 + t;
            return r < used * p.ratio;
        });
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qReady);
    };
    const unsigned char* const plane = p.cache + (((size_t)b * p.G + g) * p.pages + 2 * skip) * Q4Page<NB>::kBytes;
    auto request = [&](int c, int j) {            // rows of tile j for conversion warp c: its sixteen of keys (c < 4) or values
        const int w = c & 3;
        if (j >= tiles || 2 * j + (w >> 1) >= pages) return;
        const unsigned char* const half = plane + (size_t)(2 * j + (w >> 1)) * Q4Page<NB>::kBytes + (c >= 4 ? Q4Page<NB>::kV : 0);
        const uint32_t to = smem_u32(smem + S::kRawAt + c * S::kRaw);
        mbar_arrive_expect_tx(bar(c), S::kRaw);
        bulk_g2s(to, half + (w & 1) * (16 * Q4Page<NB>::kRow), 16 * Q4Page<NB>::kRow, bar(c));
        bulk_g2s(to + 16 * Q4Page<NB>::kRow, half + Q4Page<NB>::kKs + (w & 1) * (32 * NB), 32 * NB, bar(c));
    };
    if (warp < 4) {
        const int row = tid, token = row * inverse >> 16, head = g * p.ratio + row - token * p.ratio;
        const bool on = token < used;
        const int m = firstToken + token;
        const int last = on ? len0 + token - skip * kKT : -1;         // the row's place in the buffers, its newest key
        s_out[row] = on ? p.out + (size_t)m * p.ldo + head * HD : nullptr;
        s_stat[row] = on && p.stats != nullptr && t0 + token >= room - p.window ? m * p.H + head : -1;
        s_since[row] = 1.0f;
        if (row == 0) { s_parts = parts; s_rows = used * p.ratio; }          // the arrival for the queries publishes them
        float c = 1.0f, top = -INFINITY;          // top: the base
        float weights = 0.0f;                     // of the tiles since the last total
        if (tiles > 0) {
            queries();
            mbar_wait_long(qReady, 0, &s_abort, p.error, 349);
            __syncwarp();
            c = s_factor[row];
        }
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
        bool ok = true;
        // Totals of this warp's rows, in the rows of the output or (blocks of a cluster) the workspace: float4s i of all rows are side by side.
        auto total = [&](int i, int there, bool shared) {
            const int at = i * there + lane, r = warp * 32 + at / (HD / 4);
            return (shared ? p.totals + ((size_t)blockIdx.x * kPT + r) * HD : s_out[r]) + 4 * (at % (HD / 4));
        };
        auto add_to_totals = [&](bool fresh) {
            const float since = s_since[tid];
            const bool plain = !fresh && __all_sync(0xffffffffu, since == 1.0f);
            const int there = min(32, s_rows - warp * 32);
            const bool shared = s_parts > 1;
#pragma unroll 1
            for (int k = 0; k < HD; k += 32) {
                uint32_t o[32];
                tmem_ld32(mine + kO + k, o);
                if (lane < there)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float* const at = total(k / 4 + i, there, shared);
                        float4 v = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                        if (plain) {
                            asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
                        } else {
                            if (!fresh) {
                                const float4 w = __ldcg(reinterpret_cast<const float4*>(at));
                                v.x = fmaf(w.x, since, v.x); v.y = fmaf(w.y, since, v.y); v.z = fmaf(w.z, since, v.z); v.w = fmaf(w.w, since, v.w);
                            }
                            __stcg(reinterpret_cast<float4*>(at), v);
                        }
                    }
            }
            s_weights[tid] = fresh ? weights : fmaf(s_weights[tid], since, weights);
            weights = 0.0f;
            s_since[tid] = 1.0f;
        };
#pragma unroll 1
        for (int j = 0; j < tiles; j++) {
            if (!__all_sync(0xffffffffu, mbar_wait_long(sFull(j & 1), (j >> 1) & 1, &s_abort, p.error, 341))) ok = false;
            tc_fence_after();
            const uint32_t at = mine + (uint32_t)((j & 1) * kKT);
            if (j > 0 && j % kSegment == 0) {                            // the next product starts from zero
                if (!__all_sync(0xffffffffu, mbar_wait_long(vEmpty, (j - 1) & 1, &s_abort, p.error, 342))) ok = false;
                tc_fence_after();
                add_to_totals(j == kSegment);
            }
            const int left = last - j * kKT;                             // newest key within the tile
            const bool cut = !__all_sync(0xffffffffu, left >= kKT - 1);
            float most = -INFINITY;
            // columns are read twice, 32 a time, rather than kept: less code and registers for a load that takes 50 cycles
            auto columns = [&](int q, uint32_t (&v)[32]) {
                tmem_ld32(at + q * 32, v);
                if (cut)
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        if (k > left - q * 32) v[k] = 0xff800000u;
            };
#pragma unroll 1
            for (int q = 0; q < kKT / 32; q++) {
                uint32_t v[32];
                columns(q, v);
                float m2[2] = {most, -INFINITY};
#pragma unroll
                for (int k = 0; k < 32; k += 2) m2[(k >> 1) & 1] = max3(m2[(k >> 1) & 1], __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
                most = fmaxf(m2[0], m2[1]);
            }
            most *= c;
            const bool grown = most - top > kTop;                        // also the first keys of a row
            if (__any_sync(0xffffffffu, grown)) {
                const float now = grown ? base_of(most) : top, f = grown && top > -INFINITY ? ex2(top - now) : 1.0f;
                if (j % kSegment > 0) {
                    if (!__all_sync(0xffffffffu, mbar_wait_long(vEmpty, (j - 1) & 1, &s_abort, p.error, 342))) ok = false;
                    tc_fence_after();
#pragma unroll 1
                    for (int k = 0; k < HD; k += 32) {
                        uint32_t o[32];
                        tmem_ld32(mine + kO + k, o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st32(mine + kO + k, o);
                    }
                }
                weights *= f;
                s_since[tid] *= f;
                top = now;
            }
            const float shift = top > -INFINITY ? -top : 0.0f;           // a row without keys yet: every weight is 2^-inf
            const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift), minus = make_float2(-1.0f, -1.0f);
            float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll 1
            for (int q = 0; q < kKT / 32; q++) {
                uint32_t v[32], w[32];
                columns(q, v);
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float2 x = fma2(make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), c2, shift2);
                    const float2 e = make_float2(ex2(x.x), ex2(x.y));
                    sums = add2(sums, e);
                    // hi: the first 11 bits; the rest is exact
                    const float2 hi = make_float2(__uint_as_float(__float_as_uint(e.x) & 0xffffe000u), __uint_as_float(__float_as_uint(e.y) & 0xffffe000u));
                    const float2 lo = fma2(hi, minus, e);
                    w[k] = half2_bits(hi.x, hi.y);
                    w[16 + k] = half2_bits(lo.x, lo.y);
                }
                tmem_st32(at + q * 32, w);                               // 32 keys: sixteen columns hi, sixteen lo
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pReady(j & 1));
            weights += sums.x + sums.y;
        }
        if (tiles > 0) {
            // through shared memory (the queries and keys have been read out), so that a warp stores whole rows
            ok = __all_sync(0xffffffffu, ok && mbar_wait_long(done, 0, &s_abort, p.error, 343));
            tc_fence_after();
            float* const stage = reinterpret_cast<float*>(smem);
            const float since = s_since[tid];
            const int there = min(32, s_rows - warp * 32);
            const bool shared = s_parts > 1;
            const float sum = tiles > kSegment ? fmaf(s_weights[tid], since, weights) : weights, inv = shared ? 1.0f : 1.0f / sum;
            if (shared) s_row[row] = make_float2(top, sum);
#pragma unroll 1
            for (int k = 0; ok && k < HD; k += 32) {
                uint32_t o[32];
                tmem_ld32(mine + kO + k, o);
                if (tiles > kSegment && lane < there)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float4 w = __ldcg(reinterpret_cast<const float4*>(total(k / 4 + i, there, shared)));
                        o[4 * i] = __float_as_uint(fmaf(w.x, since, __uint_as_float(o[4 * i])));
                        o[4 * i + 1] = __float_as_uint(fmaf(w.y, since, __uint_as_float(o[4 * i + 1])));
                        o[4 * i + 2] = __float_as_uint(fmaf(w.z, since, __uint_as_float(o[4 * i + 2])));
                        o[4 * i + 3] = __float_as_uint(fmaf(w.w, since, __uint_as_float(o[4 * i + 3])));
                    }
#pragma unroll
                for (int i = 0; i < 8; i++) {     // dims 4t … 4t + 3, 16 dims on for the high nibbles
                    const int from = 8 * (i & 3) + 2 * (i >> 2);
                    *reinterpret_cast<float4*>(stage + row * PITCH + k + 4 * i) =
                        make_float4(__uint_as_float(o[from]) * inv, __uint_as_float(o[from + 4]) * inv, __uint_as_float(o[from + 1]) * inv, __uint_as_float(o[from + 5]) * inv);
                }
            }
            __syncwarp();                         // a warp stores the rows that it has staged
            const int e = lane % LPR;
            if (ok && !shared) {
#pragma unroll 8
                for (int i = lane / LPR; i < there; i += RPW)
                    *reinterpret_cast<float4*>(s_out[warp * 32 + i] + 4 * e) = *reinterpret_cast<const float4*>(stage + (warp * 32 + i) * PITCH + 4 * e);
                if (s_stat[row] >= 0) *reinterpret_cast<float2*>(p.stats + (size_t)s_stat[row] * 2) = make_float2(top, sum);
            }
        }
    } else if (warp < 12) {
        const bool value = warp >= 8;
        const int w = warp & 3, row = 16 * w + (lane & 15), t0w = lane >> 4 << 1;        // row of the tile, first of this lane's two pieces
        const unsigned char* const raw_at = smem + S::kRawAt + (warp - 4) * S::kRaw;
        unsigned char* const tile = smem + (value ? S::kVAt : S::kKAt);
        const uint32_t arrived = bar(warp - 4);
        const unsigned char* const from = plane + (size_t)(w >> 1) * Q4Page<NB>::kBytes + (value ? Q4Page<NB>::kV : 0) + (w & 1) * (16 * Q4Page<NB>::kRow);
        if (tiles > 0) queries();
        int j = 0, asked = 0;                     // asked: the last tile whose rows were
#pragma unroll 1
        for (; j < tiles; j++) {
            const bool there = 2 * j + (w >> 1) < pages;
            uint32_t words[2][NB];
            float scale[NB];
            if (there) {
                if (!__all_sync(0xffffffffu, mbar_wait_long(arrived, j & 1, &s_abort, p.error, 345))) break;
                piece_of<NB>(words[0], raw_at + Q4Page<NB>::word(lane & 15, t0w, 0));
                piece_of<NB>(words[1], raw_at + Q4Page<NB>::word(lane & 15, t0w + 1, 0));
#pragma unroll
                for (int i = 0; i < NB; i++)
                    scale[i] = __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(raw_at + 16 * Q4Page<NB>::kRow + ((lane & 15) * NB + i) * 2) << 16);
                fence_proxy_async_smem();         // the rows are read before the next copy comes over them
                __syncwarp();
                asked = j + 1;                    // everything of this tile is in registers
                if (lane == 0 && j + 1 < tiles && 2 * (j + 1) + (w >> 1) < pages) {
                    mbar_arrive_expect_tx(arrived, S::kRaw);
                    const unsigned char* const next = from + (size_t)(j + 1) * (2 * Q4Page<NB>::kBytes);
                    bulk_g2s(smem_u32(raw_at), next, 16 * Q4Page<NB>::kRow, arrived);
                    bulk_g2s(smem_u32(raw_at) + 16 * Q4Page<NB>::kRow, next + Q4Page<NB>::kKs - (w & 1) * (16 * Q4Page<NB>::kRow - 32 * NB), 32 * NB, arrived);
                }
            }
            if (j >= 1 && !__all_sync(0xffffffffu, mbar_wait_long(value ? vEmpty : kEmpty, (j - 1) & 1, &s_abort, p.error, 344))) break;
            if (there) convert_pieces<NB, kKT>(words, scale, tile, row, t0w);
            else if (value) zero_row<NB, kKT>(tile, row, t0w, t0w + 2);      // weights of 0 meet no garbage
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(value ? vFull : kFull);
        }
        if (j < tiles && 2 * min(asked, tiles - 1) + (w >> 1) < pages) wait_out(arrived, min(asked, tiles - 1) & 1);
    } else {
        // The whole warp walks the loop and one lane's predicate issues: in one lane's branch every operand would be moved into a uniform register first (70
        // cycles an MMA).  Rolled: what is issued has to come from the instruction cache in time.
        pdl_wait();
        pdl_launch_dependents();
        if (lane < 8) request(lane, 0);
        __syncwarp();
        const uint32_t lead = elect_one();
        auto waited = [&](uint32_t on, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait_long(on, parity, &s_abort, p.error, code)); };
        auto scores = [&](int j) {
            const uint32_t d = tmem + (uint32_t)((j & 1) * kKT);
            const uint64_t q0 = desc_k(base), k0 = desc_k(base + S::kKAt);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < S::kChunks; c++) {
                    const uint64_t a = q0 + (uint32_t)(((1 - h) * S::kQ + c * (kPT * 128)) >> 4), b = k0 + (uint32_t)((c * (kKT * 128)) >> 4);
#pragma unroll
                    for (int k = 0; k < (HD < 64 ? HD / 16 : 4); k++) umma_f16_by(lead, d, a + 2 * k, b + 2 * k, kIdescQK, (h | c | k) != 0);
                }
            umma_commit_by(lead, kEmpty);
            umma_commit_by(lead, sFull(j & 1));
        };
        if (tiles > 0 && waited(qReady, 0, 349) && waited(kFull, 0, 346)) {
            tc_fence_after();
            scores(0);
            int j = 0;
#pragma unroll 1
            for (; j < tiles; j++) {
                if (j + 1 < tiles) {
                    // P·V of tile j - 1 has read the buffer that the scores of j + 1 go to
                    if (j >= 1 && !waited(vEmpty, (j - 1) & 1, 350)) break;
                    if (!waited(kFull, (j + 1) & 1, 347)) break;
                    tc_fence_after();
                    scores(j + 1);
                }
                if (!waited(vFull, j & 1, 347) || !waited(pReady(j & 1), (j >> 1) & 1, 348)) break;
                tc_fence_after();
                const uint64_t v0 = desc_mn(base + S::kVAt);
                const uint32_t a = tmem + (uint32_t)((j & 1) * kKT);
#pragma unroll
                for (int k = 0; k < kKT / 16; k++) {
                    umma_f16_ta_by(lead, tmem + kO, a + (k >> 1) * 32 + (k & 1) * 8, v0 + (uint32_t)(k * 2048 >> 4), kIdescPV, (j % kSegment | k) != 0);
                    umma_f16_ta_by(lead, tmem + kO, a + (k >> 1) * 32 + 16 + (k & 1) * 8, v0 + (uint32_t)(k * 2048 >> 4), kIdescPV, 1);
                }
                umma_commit_by(lead, vEmpty);
            }
            umma_commit_by(lead, done);
            if (j < tiles) wait_out(done, 0);
        }
        __syncwarp();
    }
    if (p.splits > 1) {
        // every block of the cluster joins a part of the rows: Σ 2^(mᵢ − m)·Oᵢ over the sum of the same with the sums of weights
        __syncwarp();
        cluster_sync();
        const int parts = s_parts, all = s_rows, rank = blockIdx.x % p.splits;
        if (parts > 1 && rank < parts && !s_abort) {
            const uint32_t stage = base, state = smem_u32(s_row);
            const int r1 = all * (rank + 1) / parts, e = lane % LPR;
#pragma unroll 2
            for (int r = all * rank / parts + warp * RPW + lane / LPR; r < r1; r += (kPThreads / 32) * RPW) {
                float2 of[kMaxSplits];
                float4 o[kMaxSplits];
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kMaxSplits; i++) {
                    of[i] = make_float2(-INFINITY, 0.0f);
                    o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (i < parts) {
                        of[i] = peer_float2(state + r * 8, i);
                        o[i] = peer_float4(stage + (r * PITCH + 4 * e) * 4, i);
                    }
                    top = fmaxf(top, of[i].x);
                }
                float sum = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < kMaxSplits; i++) {
                    const float f = top > -INFINITY ? ex2(of[i].x - top) : 1.0f;      // no maximum: a row of NaN
                    sum = fmaf(of[i].y, f, sum);
                    v.x = fmaf(o[i].x, f, v.x); v.y = fmaf(o[i].y, f, v.y); v.z = fmaf(o[i].z, f, v.z); v.w = fmaf(o[i].w, f, v.w);
                }
                const float inv = 1.0f / sum;
                *reinterpret_cast<float4*>(s_out[r] + 4 * e) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                if (e == 0 && s_stat[r] >= 0) *reinterpret_cast<float2*>(p.stats + (size_t)s_stat[r] * 2) = make_float2(top, sum);
            }
        }
        __syncwarp();
        cluster_sync();                           // the rows have been read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) { tc_fence_after(); tmem_dealloc(tmem, 256); }
}

// ───────────── weights of the last tokens ─────────────
// Row i of a key/value head: its old weight and the softmax weights of the sequence's last `window` tokens.  The product is taken the other way round,
// Sᵀ = K·Qᵀ, so that a thread is a key and half of the queries and adds up its row over them in a fixed order.  A block takes 128 keys and 128 query rows
// at a time.  Bound by latency: laying the queries down, one tile after the other.
constexpr int kWThreads = 256;
template <int NB> struct WindowShape {
    static constexpr int kTile = PrefillShape<NB>::kQ;
    static constexpr int kHalvesAt = 3 * kTile;                          // Q hi, Q lo, K
    static constexpr size_t kSmem = (size_t)kHalvesAt + 4 * Q4Page<NB>::kHalf + 1024;
};
template <int NB>
__global__ void __launch_bounds__(kWThreads, 2) k_q4_window(const PrefillParams p) {
    using S = WindowShape<NB>;
    constexpr int HD = 32 * NB;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bar;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ float s_factor[kPT], s_half[kPT];  // s_half: the sums of the second half of the queries
    __shared__ float4 s_row[kPT];                 // factor, -base, 1 / sum, newest key of every query row
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, mine = tid & (kPT - 1), part = tid / kPT, g = blockIdx.y, b = blockIdx.z;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    if (tid == 0) {
        mbar_init(smem_u32(&s_bar), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // before the next kernel may come in: its blocks could hold the tensor memory until this kernel is done
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), 128);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // The kernel before has passed its own wait: all but the statistics that it writes is complete.
    bool waited = false;
    auto wait = [&]() {
        if (waited) return;
        pdl_wait();
        pdl_launch_dependents();
        waited = true;
    };
    if (p.M == 0) wait();                         // there is no such kernel then
    int first;
    const int tokens = q4_rows(__ldcg(p.starts + b), __ldcg(p.starts + b + 1), p.M, first), len = q4_int(__ldcg(p.len + b)), pos = q4_int(__ldcg(p.pos + b));
    const bool there = len >= 0 && len < p.maxSeq && pos >= 0 && pos < p.maxPos;
    const int room = q4_room(tokens, len, p.maxSeq, pos, p.maxPos), keys = there ? len + room : 0, pages = (keys + kQ4Page - 1) / kQ4Page;
    const int window = min(p.window, room), rows = window * p.ratio;
    const uint32_t tmem = s_tmem;
    unsigned char* const half = smem + S::kHalvesAt + (warp & 3) * Q4Page<NB>::kHalf;
    const unsigned char* const plane = p.cache + ((size_t)b * p.G + g) * p.pages * Q4Page<NB>::kBytes;
    auto fetch = [&](int k0) {                    // a page of a tile to two warps
        const int pg = k0 / kQ4Page + (warp & 3);
        if (k0 < keys && pg < pages)
            for (int i = part * 32 + lane; i < Q4Page<NB>::kHalf / 16; i += 64) cp_async16(half + 16 * i, plane + (size_t)pg * Q4Page<NB>::kBytes + 16 * i);
        cp_async_commit();
    };
    int phase = 0;
    if (rows > 0) fetch((int)blockIdx.x * kPT);
    for (int k0 = (int)blockIdx.x * kPT; k0 < keys; k0 += (int)gridDim.x * kPT) {
        const int key = k0 + mine;
        const size_t at = ((size_t)b * p.G + g) * p.maxSeq + key;
        const float old = part == 0 && key < len ? __ldcg(p.acc + at) : 0.0f;
        float add = 0.0f;
        if (rows > 0) {
            for (int r0 = 0; r0 < rows; r0 += kPT) {
                const int n = min(rows - r0, kPT), columns = (n + 15) & ~15;
                if (k0 == (int)blockIdx.x * kPT || rows > kPT) {         // the queries stay for all tiles if one tile holds them
                    query_rows<NB>(p, warp, kWThreads / 32, lane, smem, smem + S::kTile, s_factor, columns, [&](int i, int& qm, int& qh, int& qp) {
                        const int row = r0 + min(i, n - 1), of = row / p.ratio, token = room - window + of;
                        qm = first + token; qh = g * p.ratio + row - of * p.ratio; qp = pos + token;
                        return i < n;
                    });
                    wait();
                    __syncthreads();
                    if (part == 0) {
                        const int t = room - window + (r0 + mine) / p.ratio;
                        float2 st = make_float2(0.0f, 1.0f);
                        if (mine < n) st = __ldcg(reinterpret_cast<const float2*>(p.stats + ((size_t)(first + t) * p.H + g * p.ratio + (r0 + mine) % p.ratio) * 2));
                        s_row[mine] = make_float4(s_factor[mine], -st.x, 1.0f / st.y, __int_as_float(mine < n ? len + t : -1));
                    }
                }
                if (r0 == 0) {
                    cp_async_wait<0>();
                    __syncthreads();
                    if (k0 / kQ4Page + (warp & 3) < pages) convert_row<NB, kPT>(half, lane, smem + 2 * S::kTile, mine, 2 * part, 2 * part + 2);
                    else zero_row<NB, kPT>(smem + 2 * S::kTile, mine, 2 * part, 2 * part + 2);
                }
                fence_proxy_async_smem();
                tc_fence_before();
                __syncthreads();
                tc_fence_after();
                if (r0 == 0) fetch(k0 + (int)gridDim.x * kPT);           // everybody has read the pages
                if (warp == 0) {
                    const uint32_t lead = elect_one(), idesc = (1u << 4) | ((uint32_t)(columns >> 3) << 17) | ((uint32_t)(kPT >> 4) << 24);
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int k = 0; k < HD / 16; k++) {
                            const uint32_t o = (uint32_t)((k >> 2) * (kPT * 128) + (k & 3) * 32);
                            umma_f16_by(lead, tmem, desc_k(base + 2 * S::kTile + o), desc_k(base + (1 - h) * S::kTile + o), idesc, (h | k) != 0);
                        }
                    umma_commit_by(lead, smem_u32(&s_bar));
                }
                __syncwarp();
                const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_bar), phase & 1, &s_abort, p.error, 350));
                phase++;
                tc_fence_after();
                float sum = 0.0f;                 // of this tile, so that no chain of additions is long (9900 equal weights: off by 1.1e-5)
#pragma unroll 1
                for (int k = part * (kPT / 2); ok && k < min(n, (part + 1) * (kPT / 2)); k += 32) {
                    uint32_t v[32];
                    tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + k, v);
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const float4 q = s_row[k + i];
                        sum += key <= __float_as_int(q.w) ? ex2(fmaf(__uint_as_float(v[i]), q.x, q.y)) * q.z : 0.0f;
                    }
                }
                add += sum;
                tc_fence_before();
                __syncthreads();                  // the queries and the sums are read out
            }
            if (part == 1) s_half[mine] = add;
            __syncthreads();
        }
        wait();
        if (part == 0 && key < keys) p.accOut[at] = rows > 0 ? old + (add + s_half[mine]) : old;
    }
    wait();
    cp_async_wait<0>();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) { tc_fence_after(); tmem_dealloc(tmem, 128); }
}

// Clusters of n blocks that the device holds at once with one block to an SM.
template <int NB>
long long resident(int n) {
    static int most[kMaxSplits + 1] = {};
    if (most[n] == 0) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = n; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.gridDim = dim3(n); cfg.blockDim = dim3(kPThreads); cfg.dynamicSmemBytes = kAlone; cfg.attrs = &attr; cfg.numAttrs = 1;
        DJ_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&most[n], k_q4_prefill<NB>, &cfg));
        most[n] = std::max(most[n], 1);
    }
    return most[n];
}

struct Plan { long long blocks; int splits, least; bool alone; };
// Few blocks share their keys in clusters, as far as all are resident: a block takes 0.97 µs for a tile (64 values a row) with an SM to itself, two on
// one 1.48.  A second wave costs more than it gives (96 blocks of 300 queries before 3300 keys: 82 µs alone, 64 by twos, 69 by threes, of which 90 fit).
// Joining takes some 3 µs: four tiles to a block at least, five where two are on an SM (512 queries of 32 heads × 128: 37 µs, with fours 41).
template <int NB>
Plan plan_of(const Q4AttnArgs& a) {
    static bool attr = false;
    if (!attr) {
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_prefill<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kAlone));
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_window<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WindowShape<NB>::kSmem));
        attr = true;
    }
    const int per = kPT / (a.H / a.G);            // tokens of a tile; a sequence has at most one that is not full
    Plan plan = {(long long)a.G * ((a.M + per - 1) / per + std::min(a.B, a.M) - 1), 1, 1, false};
    plan.alone = plan.blocks <= g_num_sms;
    double best = plan.alone ? 1.0 : 1.5;
    for (int n = 2; n <= kMaxSplits; n++)
        for (int two = 0; two < 2; two++) {
            const int least = two ? 5 : 4, parts = std::min(n, a.maxSeq / (least * kKT));
            const double cost = (two ? 1.5 : 1.0) / std::max(parts, 1);
            if (parts > 1 && cost < best && plan.blocks <= (two + 1) * resident<NB>(n)) { best = cost; plan.alone = !two; plan.splits = n; plan.least = least; }
        }
    return plan;
}
Plan plan_of(const Q4AttnArgs& a) { return a.hd == 128 ? plan_of<4>(a) : a.hd == 64 ? plan_of<2>(a) : plan_of<1>(a); }

size_t stats_floats(const Q4AttnArgs& a) { return a.accOut != nullptr ? ((size_t)a.M * a.H * 2 + 3) / 4 * 4 : 0; }

template <int NB>
void prefill(PrefillParams p, const Plan& plan, cudaStream_t s) {
    p.splits = plan.splits; p.least = plan.least;
    // a grid that gives every block an SM of its own asks for so much shared memory that it gets one (blocks are dealt out two to an SM otherwise)
    const size_t smem = plan.alone ? kAlone : PrefillShape<NB>::kSmem;
    if (p.M > 0) launch_k_cluster(k_q4_prefill<NB>, dim3((unsigned)(plan.blocks * p.splits)), dim3(kPThreads), smem, s, dim3(p.splits), p);
    // a block's queries serve all its key tiles: about two blocks per SM
    const int tiles = (p.maxSeq + kPT - 1) / kPT, share = std::max(1, 2 * g_num_sms / std::max(1, p.G * p.B));
    if (p.accOut != nullptr) launch_k(k_q4_window<NB>, dim3(std::min(tiles, share), p.G, p.B), dim3(kWThreads), WindowShape<NB>::kSmem, s, true, p);
}

}  // namespace

size_t q4_attn_ws_floats(const Q4AttnArgs& a) {
    const Plan plan = plan_of(a);
    return stats_floats(a) + (a.M > 0 && plan.splits > 1 && a.maxSeq > kSegment * kKT ? (size_t)plan.blocks * plan.splits * kPT * a.hd : 0);
}

void launch_q4_attn(const Q4AttnArgs& a, cudaStream_t s) {
    const PrefillParams p = {a.qkv, a.q_off, a.ld, a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.starts, a.len, a.pos, a.cosT, a.sinT, a.maxPos, a.out, a.ldo,
                             a.B, a.H, a.G, a.H / a.G, a.M, (float)(1.0 / std::sqrt((double)a.hd) * 1.4426950408889634), a.accOut != nullptr ? a.ws : nullptr, a.window,
                             a.acc, a.accOut, g_dev_error, a.ws + stats_floats(a), 1, 1};
    const Plan plan = plan_of(a);
    if (a.M > 0) launch_q4_append(a, 1, s);
    if (a.hd == 128) prefill<4>(p, plan, s); else if (a.hd == 64) prefill<2>(p, plan, s); else prefill<1>(p, plan, s);
}

}  // namespace dj
