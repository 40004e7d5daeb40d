// Packed prompts over the 4-bit cache on the 5th-generation tensor cores.
//
// A block takes 128 query rows of one key/value head: 128 / R consecutive tokens of one sequence times the R query heads that share the head, so that a
// key or value is brought and converted once for all of them.  It walks the cached rows in tiles of 128:
//   S = Q·Kᵀ    Q in fp16 halves hi + lo of the rotated row times a power of two (22 bits); a stored key, code · scale, is exact in fp16: two MMAs
//   P = 2^(S·c − m) per row, in halves hi + lo again, written over S in tensor memory, from where it is the A operand of
//   O += P·V    with O in tensor memory as well
//   warps 0-7   two threads to a row: running maximum and sum of the softmax in fp32, no exchange between lanes.  O is multiplied by the change of the
//               maximum only when that grew by more than 2^8: until then P is larger than one, which fp16 and the fp32 sums have room for
//   warps 8-15  two warps are a page: 4-bit codes → fp16 tiles with 128-byte swizzle, keys a tile ahead of the values
//   warp 16     one thread brings the pages' halves with bulk copies into a ring
//   warp 17     one thread issues the MMAs: Q·K of the next tile before P·V of this one, so that the softmax never waits for them
// Tensor memory: three S/P buffers of 128 columns and O.  Every wait is bounded (codes 341-349 in the device error word).
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "q4_cache.cuh"
#include "tc_common.cuh"
#include <cuda_fp16.h>

namespace dj {
namespace {

constexpr int kPT = 128;                          // query rows and keys of a tile
constexpr int kPThreads = 576;                    // warps: 8 softmax, 8 conversion, copies, MMAs
constexpr int kPRing = 3;                         // ring stages: the K or the V halves of a tile's four pages

struct PrefillParams {
    const float* qkv; int q_off, ld;
    const unsigned char* cache; int maxSeq, pages;
    const float* starts; const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    float* out; int ldo; int B, H, G, ratio, M; float scale;            // scale: 1/sqrt(hd) · log2(e)
    float* stats; int window;                     // [M][H][2] maximum (log2) and sum of the last `window` tokens' rows, or null
    const float* acc; float* accOut;
    int* error;
};

template <int NB> struct PrefillShape {
    static constexpr int HD = 32 * NB, kChunks = (HD + 63) / 64, kTile = kChunks * kPT * 128;      // bytes of 128 rows in 128-byte pieces
    static constexpr int kStage = 4 * Q4Page<NB>::kHalf;
    static constexpr int kRingAt = 6 * kTile;                            // Q hi, Q lo, K × 2, V × 2
    static constexpr size_t kUsed = (size_t)kRingAt + kPRing * kStage + 1024;
    static constexpr size_t kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;      // one block per SM: it holds all tensor memory
};

// K-major, 128-byte swizzle: 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3fff) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// MN-major: 64 dims to a 128-byte row, 8-key groups 1024 bytes apart, the next 64 dims 128 rows on
__device__ __forceinline__ uint64_t desc_mn(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3fff) | ((uint64_t)(kPT * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
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
template <int NB, bool WIDE>
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
            *reinterpret_cast<uint4*>(tile + (j >> 1) * (kPT * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                make_uint4(half_of(w[j] << 6, scale[j], off[j], WIDE), half_of(w[j] << 2, scale[j], off[j], WIDE), half_of(w[j] >> 2, scale[j], off[j], WIDE),
                           half_of(w[j] >> 6, scale[j], off[j], WIDE));
        }
    }
}
// Row `lane` of a page's K or V half, its words (t0 … t1 - 1, j) → row `row` of an fp16 tile.
template <int NB>
__device__ __forceinline__ void convert_row(const unsigned char* half, int lane, unsigned char* tile, int row, int t0, int t1) {
    __half2 scale[NB];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        const float s = __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(half + Q4Page<NB>::kKs + (lane * NB + j) * 2) << 16);
        most = fmaxf(most, s);
        scale[j] = __float2half2_rn(s);
    }
    if (__any_sync(0xffffffffu, most > 2048.0f)) convert_words<NB, true>(half, lane, tile, row, scale, t0, t1);
    else convert_words<NB, false>(half, lane, tile, row, scale, t0, t1);
}
template <int NB>
__device__ __forceinline__ void zero_row(unsigned char* tile, int row, int t0, int t1) {
#pragma unroll 1
    for (int c = 0; c < 4 * NB; c++)
        if ((c & 3) >= t0 && (c & 3) < t1) *reinterpret_cast<uint4*>(tile + (c >> 3) * (kPT * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
}

// Query rows of a tile, rotated, in halves of fp16 times a power of two → tiles hi and lo, a row to 8·NB lanes of four values each; `place(row, m, head, position)` says
// which one row `row` is (false: zeros).  factors[row] makes a sum of products a score in log2 units (NaN where the row holds an infinity or a NaN).
template <int NB, typename Place>
__device__ __forceinline__ void query_rows(const PrefillParams& p, int warp, int warps, int lane, unsigned char* hi, unsigned char* lo, float* factors, Place place) {
    constexpr int HD = 32 * NB, LPR = 8 * NB, RPW = 32 / LPR;
    const int e = lane % LPR;
    // this lane's dims 4e … 4e + 3 in the tiles' order: (0, 2) and (1, 3), eight bytes apart
    const int piece = (e >> 3) * 4 + (e & 3), at = (piece >> 3) * (kPT * 128) + (e & 4);
#pragma unroll 4
    for (int r = warp * RPW + lane / LPR; r < kPT; r += warps * RPW) {
        int m, head, position;
        const bool on = place(r, m, head, position);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (on) {
            const size_t tab = (size_t)position * (HD / 2) + 2 * e;
            x = q4_rotate(*reinterpret_cast<const float4*>(p.qkv + (size_t)m * p.ld + p.q_off + head * HD + 4 * e), *reinterpret_cast<const float2*>(p.cosT + tab),
                          *reinterpret_cast<const float2*>(p.sinT + tab));
        }
        float most = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))), bad = (x.x + x.y + x.z + x.w) * 0.0f;
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) { most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o)); bad += __shfl_xor_sync(0xffffffffu, bad, o); }
        // the largest value comes to 256 … 512
        most = fmaxf(most, 7.8886091e-31f);
        const int bits = __float_as_int(most) & 0x7f800000;
        const bool fine = bad == 0.0f && most < 1e30f;
        const float mul = fine ? __int_as_float(0x7f000000 - bits) * 256.0f : 0.0f;
        if (!fine) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        uint2 h, l;
        split_half(x.x * mul, x.z * mul, h.x, l.x);
        split_half(x.y * mul, x.w * mul, h.y, l.y);
        const int to = at + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint32_t*>(hi + to) = h.x; *reinterpret_cast<uint32_t*>(hi + to + 8) = h.y;
        *reinterpret_cast<uint32_t*>(lo + to) = l.x; *reinterpret_cast<uint32_t*>(lo + to + 8) = l.y;
        if (e == 0) factors[r] = fine ? __int_as_float(bits) * (1.0f / 256.0f) * p.scale : __int_as_float(0x7fc00000);
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

// Sequence and first token of query tile `tile`, the last tile of a sequence first; whole warps call it.
__device__ __forceinline__ bool tile_of(const PrefillParams& p, int tile, int tokensPerTile, int lane, int& b, int& first, int& tokens, int& t0) {
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        int from = 0, n = 0;
        if (b0 + lane < p.B) {
            from = max(0, (int)p.starts[b0 + lane]);
            n = max(0, min(p.M, (int)p.starts[b0 + lane + 1]) - from);
        }
        const int tiles = (n + tokensPerTile - 1) / tokensPerTile;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < upto);
        if (hit) {
            const int l = __ffs(hit) - 1;
            b = b0 + l;
            first = __shfl_sync(0xffffffffu, from, l);
            tokens = __shfl_sync(0xffffffffu, n, l);
            t0 = (__shfl_sync(0xffffffffu, upto, l) - 1 - tile) * tokensPerTile;
            return true;
        }
        tile -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <int NB>
__global__ void __launch_bounds__(kPThreads, 1) k_q4_prefill(const PrefillParams p) {
    using S = PrefillShape<NB>;
    constexpr int HD = S::HD;
    constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kPT >> 3) << 17) | ((uint32_t)(kPT >> 4) << 24);      // fp16 × fp16 → fp32
    constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kPT >> 4) << 24);      // B MN-major
    constexpr uint32_t kO = 3 * kPT;              // O's first column
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bar[2 * kPRing + 14];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ float s_max[2][2][kPT], s_factor[kPT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
    auto ringFull = [&](int s) { return bar(s); };
    auto ringEmpty = [&](int s) { return bar(kPRing + s); };
    auto kEmpty = [&](int s) { return bar(2 * kPRing + s); };           // Q·K of a tile is done
    auto vFull = [&](int s) { return bar(2 * kPRing + 2 + s); };         // the values of a tile stand, and so do the keys of the next one
    auto vEmpty = [&](int s) { return bar(2 * kPRing + 4 + s); };        // P·V of a tile is done
    auto sFull = [&](int s) { return bar(2 * kPRing + 6 + s); };
    auto pReady = [&](int s) { return bar(2 * kPRing + 9 + s); };
    const uint32_t qReady = bar(2 * kPRing + 12), firstKeys = bar(2 * kPRing + 13);
    if (tid == 0) {
        for (int s = 0; s < kPRing; s++) { mbar_init(ringFull(s), 1); mbar_init(ringEmpty(s), 8); }
        for (int s = 0; s < 2; s++) { mbar_init(kEmpty(s), 1); mbar_init(vFull(s), 8); mbar_init(vEmpty(s), 1); }
        for (int s = 0; s < 3; s++) { mbar_init(sFull(s), 1); mbar_init(pReady(s), 8); }
        mbar_init(qReady, 8);
        mbar_init(firstKeys, 8);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) tmem_alloc(smem_u32(&s_tmem), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_wait();
    pdl_launch_dependents();

    const int g = blockIdx.x % p.G, tokensPerTile = kPT / p.ratio;
    int b = 0, first = 0, tokens = 0, t0 = 0, len = 0, pos = 0, room = 0;
    if (tile_of(p, blockIdx.x / p.G, tokensPerTile, lane, b, first, tokens, t0)) {
        len = (int)p.len[b]; pos = (int)p.pos[b];
        room = q4_room(tokens, len, p.maxSeq, pos, p.maxPos);
    }
    const int used = max(0, min(tokensPerTile, room - t0));              // tokens of this tile
    const int keys = used > 0 ? len + t0 + used : 0, tiles = (keys + kPT - 1) / kPT, pages = (keys + kQ4Page - 1) / kQ4Page;

    if (warp < 8) {
        // two threads to a row, 64 keys of a tile each: warps w and w + 4 exchange what they find through shared memory
        const int part = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, token = row / p.ratio, head = g * p.ratio + row % p.ratio;
        const bool on = token < used;
        const int m = first + t0 + token, last = on ? len + t0 + token : -1;      // the row's place in the buffers, its newest key
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); };
        float c = 1.0f, top = -INFINITY;
        float2 sums = make_float2(0.0f, 0.0f);
        if (tiles > 0) {
            query_rows<NB>(p, warp, 8, lane, smem, smem + S::kTile, s_factor, [&](int r, int& qm, int& qh, int& qp) {
                const int t = r / p.ratio;
                qm = first + t0 + t; qh = g * p.ratio + r - t * p.ratio; qp = pos + t0 + t;
                return t < used;
            });
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(qReady);
            asm volatile("bar.sync 5, 256;" ::: "memory");
            c = s_factor[row];
        }
        const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
        bool ok = true;
        for (int j = 0; j < tiles; j++) {
            if (!__all_sync(0xffffffffu, mbar_wait(sFull(j % 3), (j / 3) & 1, &s_abort, p.error, 341))) ok = false;
            tc_fence_after();
            const uint32_t at = mine + (uint32_t)(j % 3 * kPT + part * 64);
            const int left = last - j * kPT - part * 64;                 // newest key within these 64
            const bool cut = !__all_sync(0xffffffffu, left >= 63);
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
            for (int q = 0; q < 2; q++) {
                uint32_t v[32];
                columns(q, v);
                float m2[2] = {most, -INFINITY};
#pragma unroll
                for (int k = 0; k < 32; k += 2) m2[(k >> 1) & 1] = max3(m2[(k >> 1) & 1], __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
                most = fmaxf(m2[0], m2[1]);
            }
            most *= c;
            s_max[j & 1][part][row] = most;
            meet();
            most = fmaxf(most, s_max[j & 1][1 - part][row]);
            const bool grown = most > top + 8.0f;                        // also the first keys of a row
            if (__any_sync(0xffffffffu, grown)) {                        // both warps of a row come to the same
                const float now = grown ? most : top, f = grown && top > -INFINITY ? ex2(top - now) : 1.0f;
                if (j > 0) {
                    if (!__all_sync(0xffffffffu, mbar_wait(vEmpty((j - 1) & 1), ((j - 1) >> 1) & 1, &s_abort, p.error, 342))) ok = false;
                    tc_fence_after();
#pragma unroll 1
                    for (int k = 32 * part; k < HD; k += 64) {
                        uint32_t o[32];
                        tmem_ld32(mine + kO + k, o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st32(mine + kO + k, o);
                    }
                }
                sums.x *= f; sums.y *= f;
                top = now;
            }
            const float shift = top > -INFINITY ? -top : 0.0f;           // a row without keys yet: every weight is 2^-inf
            const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift), minus = make_float2(-1.0f, -1.0f);
#pragma unroll 1
            for (int q = 0; q < 2; q++) {
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
            if (lane == 0) mbar_arrive(pReady(j % 3));
        }
        float sum = sums.x + sums.y;
        if (tiles > 0) {
            s_max[tiles & 1][part][row] = sum;
            meet();
            sum += s_max[tiles & 1][1 - part][row];
        }
        if (tiles > 0) {
            // through shared memory (the queries and keys have been read out), so that a warp stores whole rows
            ok = __all_sync(0xffffffffu, ok && mbar_wait(vEmpty((tiles - 1) & 1), ((tiles - 1) >> 1) & 1, &s_abort, p.error, 343));
            tc_fence_after();
            const float inv = 1.0f / sum;
            constexpr int PITCH = HD + 4, LPR = 8 * NB, RPW = 32 / LPR;
            float* const stage = reinterpret_cast<float*>(smem);
#pragma unroll 1
            for (int k = 32 * part; ok && k < HD; k += 64) {
                uint32_t o[32];
                tmem_ld32(mine + kO + k, o);
#pragma unroll
                for (int i = 0; i < 8; i++) {     // dims 4t … 4t + 3, 16 dims on for the high nibbles
                    const int from = 8 * (i & 3) + 2 * (i >> 2);
                    *reinterpret_cast<float4*>(stage + row * PITCH + k + 4 * i) =
                        make_float4(__uint_as_float(o[from]) * inv, __uint_as_float(o[from + 4]) * inv, __uint_as_float(o[from + 1]) * inv, __uint_as_float(o[from + 5]) * inv);
                }
            }
            asm volatile("bar.sync 5, 256;" ::: "memory");
            for (int r = warp * RPW + lane / LPR; ok && r < used * p.ratio; r += 8 * RPW) {
                const int t = r / p.ratio, e = lane % LPR;
                *reinterpret_cast<float4*>(p.out + (size_t)(first + t0 + t) * p.ldo + (g * p.ratio + r - t * p.ratio) * HD + 4 * e) =
                    *reinterpret_cast<const float4*>(stage + r * PITCH + 4 * e);
            }
            if (part == 0 && on && p.stats != nullptr && t0 + token >= room - p.window)
                *reinterpret_cast<float2*>(p.stats + ((size_t)m * p.H + head) * 2) = make_float2(top, sum);
        }
    } else if (warp < 16) {
        const int w = warp & 3, t0 = (warp - 8) >> 2 << 1;               // page of the tile, half of a row's words
        bool ok = true;
        int item = 0;
#pragma unroll 1
        for (int i = 0; i < 2 * tiles && ok; i++) {                      // K 0, K 1, V 0, K 2, V 1, …, V tiles - 1
            const bool value = i > 0 && (i % 2 == 0 || i == 2 * tiles - 1);
            const int j = i == 0 ? 0 : value ? (i - 1) / 2 : (i + 1) / 2;
            if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(value ? vEmpty(j & 1) : kEmpty(j & 1), ((j >> 1) - 1) & 1, &s_abort, p.error, 344))) break;
            if (!__all_sync(0xffffffffu, mbar_wait(ringFull(item % kPRing), (item / kPRing) & 1, &s_abort, p.error, 345))) break;
            unsigned char* const tile = smem + (value ? 4 + (j & 1) : 2 + (j & 1)) * S::kTile;
            if (4 * j + w < pages) convert_row<NB>(smem + S::kRingAt + item % kPRing * S::kStage + w * Q4Page<NB>::kHalf, lane, tile, 32 * w + lane, t0, t0 + 2);
            else if (value) zero_row<NB>(tile, 32 * w + lane, t0, t0 + 2);      // weights of 0 meet no garbage
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(ringEmpty(item % kPRing));
                if (value) mbar_arrive(vFull(j & 1));
                else if (j == 0) mbar_arrive(firstKeys);
            }
            item++;
        }
    } else if (warp == 16) {
        if (lane == 0) {
            const unsigned char* const plane = p.cache + ((size_t)b * p.G + g) * p.pages * Q4Page<NB>::kBytes;
            int item = 0;
            bool ok = true;
            auto bring = [&](int j, bool value) {
                const int s = item % kPRing, n = min(4, pages - 4 * j);
                if (item >= kPRing && !mbar_wait(ringEmpty(s), (item / kPRing - 1) & 1, &s_abort, p.error, 346)) return false;
                mbar_arrive_expect_tx(ringFull(s), n * Q4Page<NB>::kHalf);
                for (int w = 0; w < n; w++)
                    bulk_g2s(base + S::kRingAt + s * S::kStage + w * Q4Page<NB>::kHalf, plane + (size_t)(4 * j + w) * Q4Page<NB>::kBytes + (value ? Q4Page<NB>::kV : 0),
                             Q4Page<NB>::kHalf, ringFull(s));
                item++;
                return true;
            };
            for (int j = 0; j <= tiles && ok; j++) {
                if (j < tiles) ok = bring(j, false);
                if (ok && j > 0) ok = bring(j - 1, true);
            }
            if (!ok)                              // a wait ran out: let the copies in flight land before the block goes
                for (int back = 1; back <= kPRing && back <= item; back++)
                    for (unsigned n = 0; n < (1u << 16) && !mbar_try_wait(ringFull((item - back) % kPRing), ((item - back) / kPRing) & 1); n++) {}
        }
        __syncwarp();
    } else {
        if (lane == 0 && tiles > 0) {
            // rolled: what one thread issues has to come from the instruction cache in time
            auto scores = [&](int j) {
                const uint32_t d = tmem + (uint32_t)(j % 3 * kPT);
                const uint64_t q0 = desc_k(base), k0 = desc_k(base + (2 + (j & 1)) * S::kTile);
#pragma unroll 1
                for (int h = 0; h < 2; h++)
#pragma unroll 1
                    for (int c = 0; c < S::kChunks; c++) {
                        const uint64_t a = q0 + (uint32_t)((h * S::kTile + c * (kPT * 128)) >> 4), b = k0 + (uint32_t)((c * (kPT * 128)) >> 4);
#pragma unroll
                        for (int k = 0; k < (HD < 64 ? HD / 16 : 4); k++) umma_f16(d, a + 2 * k, b + 2 * k, kIdescQK, (h | c | k) != 0);
                    }
                umma_commit(kEmpty(j & 1));
                umma_commit(sFull(j % 3));
            };
            if (mbar_wait(qReady, 0, &s_abort, p.error, 349) && mbar_wait(firstKeys, 0, &s_abort, p.error, 346)) {
                tc_fence_after();
                scores(0);
#pragma unroll 1
                for (int j = 0; j < tiles; j++) {
                    // values of tile j: the keys of j + 1 were converted before them, and P·V of j - 2, which read the scores' buffer of j + 1, was
                    // done before they came
                    if (!mbar_wait(vFull(j & 1), (j >> 1) & 1, &s_abort, p.error, 347)) break;
                    tc_fence_after();
                    if (j + 1 < tiles) scores(j + 1);
                    if (!mbar_wait(pReady(j % 3), (j / 3) & 1, &s_abort, p.error, 348)) break;
                    tc_fence_after();
                    const uint64_t v0 = desc_mn(base + (4 + (j & 1)) * S::kTile);
                    const uint32_t a = tmem + (uint32_t)(j % 3 * kPT);
#pragma unroll 2
                    for (int k = 0; k < kPT / 16; k++) {
                        umma_f16_ta(tmem + kO, a + (k >> 1) * 32 + (k & 1) * 8, v0 + (uint32_t)(k * 2048 >> 4), kIdescPV, (j | k) != 0);
                        umma_f16_ta(tmem + kO, a + (k >> 1) * 32 + 16 + (k & 1) * 8, v0 + (uint32_t)(k * 2048 >> 4), kIdescPV, 1);
                    }
                    umma_commit(vEmpty(j & 1));
                }
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// ───────────── weights of the last tokens ─────────────
// Row i of a key/value head: its old weight and the softmax weights of the sequence's last `window` tokens.  The product is taken the other way round,
// Sᵀ = K·Qᵀ, so that a thread is a key and adds up its row over the queries in a fixed order.  A block takes 128 keys and 128 query rows at a time.
constexpr int kWThreads = 128;
template <int NB> struct WindowShape {
    static constexpr int kTile = PrefillShape<NB>::kTile;
    static constexpr int kHalvesAt = 3 * kTile;                          // Q hi, Q lo, K
    static constexpr size_t kSmem = (size_t)kHalvesAt + 4 * Q4Page<NB>::kHalf + 1024;
};
template <int NB>
__global__ void __launch_bounds__(kWThreads) k_q4_window(const PrefillParams p) {
    using S = WindowShape<NB>;
    constexpr int HD = 32 * NB;
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kPT >> 3) << 17) | ((uint32_t)(kPT >> 4) << 24);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long s_bar;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ float s_factor[kPT];
    __shared__ float4 s_row[kPT];                 // factor, maximum, 1 / sum, newest key of every query row
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = blockIdx.y, b = blockIdx.z;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    if (tid == 0) {
        mbar_init(smem_u32(&s_bar), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // before the next kernel may come in: its blocks could hold the tensor memory until this kernel is done
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), 128);
    pdl_wait();
    pdl_launch_dependents();
    const int first = max(0, (int)p.starts[b]), tokens = max(0, min(p.M, (int)p.starts[b + 1]) - first), len = (int)p.len[b], pos = (int)p.pos[b];
    const bool there = len >= 0 && len < p.maxSeq && pos >= 0 && pos < p.maxPos;
    const int room = q4_room(tokens, len, p.maxSeq, pos, p.maxPos), keys = there ? len + room : 0, k0 = blockIdx.x * kPT, key = k0 + tid;
    const int window = min(p.window, room), rows = k0 < keys ? window * p.ratio : 0;
    const size_t at = ((size_t)b * p.G + g) * p.maxSeq + key;
    float add = 0.0f;
    if (rows > 0) {
        // the tile's keys: a warp is a page
        const int pages = (keys + kQ4Page - 1) / kQ4Page, pg = k0 / kQ4Page + warp;
        unsigned char* const half = smem + S::kHalvesAt + warp * Q4Page<NB>::kHalf;
        if (pg < pages) {
            const uint4* const from = reinterpret_cast<const uint4*>(p.cache + (((size_t)b * p.G + g) * p.pages + pg) * Q4Page<NB>::kBytes);
            for (int i = lane; i < Q4Page<NB>::kHalf / 16; i += 32) reinterpret_cast<uint4*>(half)[i] = from[i];
            __syncwarp();
            convert_row<NB>(half, lane, smem + 2 * S::kTile, tid, 0, 4);
        } else zero_row<NB>(smem + 2 * S::kTile, tid, 0, 4);
        int phase = 0;
        for (int r0 = 0; r0 < rows; r0 += kPT) {
            const int r = r0 + tid, t = room - window + r / p.ratio, head = g * p.ratio + r % p.ratio, m = first + t;
            const bool on = r < rows;
            query_rows<NB>(p, warp, 4, lane, smem, smem + S::kTile, s_factor, [&](int i, int& qm, int& qh, int& qp) {
                const int of = (r0 + i) / p.ratio, token = room - window + of;
                qm = first + token; qh = g * p.ratio + r0 + i - of * p.ratio; qp = pos + token;
                return r0 + i < rows;
            });
            __syncthreads();
            float2 st = make_float2(0.0f, 1.0f);
            if (on) st = *reinterpret_cast<const float2*>(p.stats + ((size_t)m * p.H + head) * 2);
            s_row[tid] = make_float4(s_factor[tid], -st.x, 1.0f / st.y, __int_as_float(on ? len + t : -1));
            fence_proxy_async_smem();
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
            const uint32_t tmem = s_tmem;
            if (tid == 0) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint32_t o = (uint32_t)((k >> 2) * (kPT * 128) + (k & 3) * 32);
                        umma_f16(tmem, desc_k(base + 2 * S::kTile + o), desc_k(base + h * S::kTile + o), kIdesc, (h | k) != 0);
                    }
                umma_commit(smem_u32(&s_bar));
            }
            __syncwarp();
            const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_bar), phase & 1, &s_abort, p.error, 350));
            phase++;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; ok && k < kPT && r0 + k < rows; k += 32) {
                uint32_t v[32];
                tmem_ld32(tmem + ((uint32_t)(warp * 32) << 16) + k, v);
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const float4 q = s_row[k + i];
                    add += key <= __float_as_int(q.w) ? ex2(fmaf(__uint_as_float(v[i]), q.x, q.y)) * q.z : 0.0f;
                }
            }
            tc_fence_before();
            __syncthreads();                      // the queries and the sums are read out
        }
    }
    if (key < keys) p.accOut[at] = (key < len ? p.acc[at] : 0.0f) + add;
    tc_fence_before();
    __syncthreads();
    if (warp == 0) { tc_fence_after(); tmem_dealloc(s_tmem, 128); }
}

template <int NB>
void prefill(const PrefillParams& p, cudaStream_t s) {
    static bool attr = false;
    if (!attr) {
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_prefill<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrefillShape<NB>::kSmem));
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_window<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WindowShape<NB>::kSmem));
        attr = true;
    }
    const int per = kPT / p.ratio;                // tokens of a tile; a sequence has at most one that is not full
    if (p.M > 0) launch_k(k_q4_prefill<NB>, dim3(p.G * ((p.M + per - 1) / per + std::min(p.B, p.M) - 1)), dim3(kPThreads), PrefillShape<NB>::kSmem, s, true, p);
    if (p.accOut != nullptr) launch_k(k_q4_window<NB>, dim3((p.maxSeq + kPT - 1) / kPT, p.G, p.B), dim3(kWThreads), WindowShape<NB>::kSmem, s, true, p);
}

}  // namespace

size_t q4_attn_ws_floats(const Q4AttnArgs& a) { return a.accOut != nullptr ? (size_t)a.M * a.H * 2 : 0; }

void launch_q4_attn(const Q4AttnArgs& a, cudaStream_t s) {
    PrefillParams p = {a.qkv, a.q_off, a.ld, a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.starts, a.len, a.pos, a.cosT, a.sinT, a.maxPos, a.out, a.ldo,
                       a.B, a.H, a.G, a.H / a.G, a.M, (float)(1.0 / std::sqrt((double)a.hd) * 1.4426950408889634), a.accOut != nullptr ? a.ws : nullptr, a.window,
                       a.acc, a.accOut, g_dev_error};
    if (a.M > 0) launch_q4_append(a, 1, s);
    if (a.hd == 128) prefill<4>(p, s); else if (a.hd == 64) prefill<2>(p, s); else prefill<1>(p, s);
}

}  // namespace dj
