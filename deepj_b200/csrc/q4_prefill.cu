// Packed prompts over the 4-bit cache on the 5th-generation tensor cores.
//
// A block takes 128 query rows of one key/value head: 128 / R consecutive tokens of one sequence times the R query heads that share the head, so that a
// key or value is brought and converted once for all of them.  It walks the cached rows in tiles of 128:
//   S = Q·Kᵀ    Q in fp16 halves hi + lo of the rotated row times a power of two (22 bits); a stored key, code · scale, is exact in fp16: two MMAs
//   P = 2^(S·c − m) per row, in halves hi + lo again, written over S in tensor memory, from where it is the A operand of
//   O += P·V    with O in tensor memory as well
//   warps 0-7   two threads to a row: running maximum and sum of the softmax in fp32, no exchange between lanes.  O is multiplied by the change of the
//               maximum only when that grew by more than 2^8: until then P is larger than one, which fp16 and the fp32 sums have room for
//   warps 8-11  a warp is a page: 4-bit codes → fp16 tiles with 128-byte swizzle, keys a tile ahead of the values
//   warp 12     one thread brings the pages' halves with bulk copies into a ring
//   warp 13     one thread issues the MMAs: Q·K of the next tile before P·V of this one, so that the softmax never waits for them
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
constexpr int kPThreads = 448;                    // warps: 8 softmax, 4 conversion, copies, MMAs
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

// Four codes in the low nibbles of a word's bytes, sign bits flipped (code + 8) → four fp16 values: 1024 + 8 + code, minus 1032, times the scale; all exact.
__device__ __forceinline__ uint2 codes_to_half(uint32_t nibbles, __half2 scale) {
    const uint32_t a = __byte_perm(nibbles, 0x64646464u, 0x4140), b = __byte_perm(nibbles, 0x64646464u, 0x4342);
    const __half2 off = __float2half2_rn(1032.0f);
    const __half2 x = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&a), off), scale), y = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&b), off), scale);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// Row `lane` of a page's K or V half → row `row` of an fp16 tile, 16 bytes (8 dims) a time.
template <int NB>
__device__ __forceinline__ void convert_row(const unsigned char* half, int lane, unsigned char* tile, int row) {
    __half2 scale[NB];
#pragma unroll
    for (int j = 0; j < NB; j++)
        scale[j] = __float2half2_rn(__uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(half + Q4Page<NB>::kKs + (lane * NB + j) * 2) << 16));
#pragma unroll 1
    for (int u = 0; u < 2; u++) {                 // rolled: the roles of a block run side by side and share the instruction cache
        uint32_t w[2][NB];
        piece_of<NB>(w[0], half + Q4Page<NB>::word(lane, 2 * u, 0));
        piece_of<NB>(w[1], half + Q4Page<NB>::word(lane, 2 * u + 1, 0));
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t a = ((w[0][j] >> (4 * x)) & 0x0f0f0f0fu) ^ 0x08080808u, b = ((w[1][j] >> (4 * x)) & 0x0f0f0f0fu) ^ 0x08080808u;
                const uint2 lo = codes_to_half(a, scale[j]), hi = codes_to_half(b, scale[j]);
                const int c = 4 * j + 2 * x + u;
                *reinterpret_cast<uint4*>(tile + (c >> 3) * (kPT * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
    }
}
template <int NB>
__device__ __forceinline__ void zero_row(unsigned char* tile, int row) {
#pragma unroll
    for (int c = 0; c < 4 * NB; c++) *reinterpret_cast<uint4*>(tile + (c >> 3) * (kPT * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
}

// A query row, rotated at `position`, in halves of fp16 times a power of two → tile row `row`; returns the factor that makes a sum of products a score
// in log2 units (NaN where the row holds an infinity or a NaN).
template <int NB>
__device__ __forceinline__ float query_row(const PrefillParams& p, int m, int head, int position, bool on, unsigned char* hi, unsigned char* lo, int row) {
    constexpr int HD = 32 * NB;
    float4 x[HD / 4];
    const float* const q = p.qkv + (size_t)m * p.ld + p.q_off + head * HD;
    const float* const cs = p.cosT + (size_t)position * (HD / 2);
    const float* const sn = p.sinT + (size_t)position * (HD / 2);
    float most = 0.0f, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 4; i++) {
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (on) x[i] = q4_rotate(*reinterpret_cast<const float4*>(q + 4 * i), *reinterpret_cast<const float2*>(cs + 2 * i), *reinterpret_cast<const float2*>(sn + 2 * i));
    }
#pragma unroll
    for (int i = 0; i < HD / 4; i++) {
        most = fmaxf(most, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        bad += (x[i].x + x[i].y + x[i].z + x[i].w) * 0.0f;
    }
    // the largest value comes to 256 … 512
    const bool some = most > 7.8886091e-31f && most < 1e30f;
    const int bits = some ? __float_as_int(most) & 0x7f800000 : 0x3f800000;
    const float mul = bad == 0.0f && some ? __int_as_float(0x7f000000 - bits) * 256.0f : 0.0f;
#pragma unroll
    for (int c = 0; c < HD / 8; c++) {
        const float4 a = x[2 * c], b = x[2 * c + 1];
        uint4 h, l;
        split_half(a.x * mul, a.y * mul, h.x, l.x); split_half(a.z * mul, a.w * mul, h.y, l.y);
        split_half(b.x * mul, b.y * mul, h.z, l.z); split_half(b.z * mul, b.w * mul, h.w, l.w);
        if (mul == 0.0f) h = l = make_uint4(0, 0, 0, 0);
        const int at = (c >> 3) * (kPT * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(hi + at) = h;
        *reinterpret_cast<uint4*>(lo + at) = l;
    }
    return __int_as_float(bits) * (1.0f / 256.0f) * p.scale + (some || most == 0.0f || bad != 0.0f ? bad : most < 1.0f ? 0.0f : __int_as_float(0x7fc00000));
}

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
    __shared__ __align__(8) unsigned long long s_bar[2 * kPRing + 8 + 6 + 1];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ float s_max[2][kPT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
    auto ringFull = [&](int s) { return bar(s); };
    auto ringEmpty = [&](int s) { return bar(kPRing + s); };
    auto kFull = [&](int s) { return bar(2 * kPRing + s); };
    auto kEmpty = [&](int s) { return bar(2 * kPRing + 2 + s); };
    auto vFull = [&](int s) { return bar(2 * kPRing + 4 + s); };
    auto vEmpty = [&](int s) { return bar(2 * kPRing + 6 + s); };        // P·V of a tile is done
    auto sFull = [&](int s) { return bar(2 * kPRing + 8 + s); };
    auto pReady = [&](int s) { return bar(2 * kPRing + 11 + s); };
    const uint32_t qReady = bar(2 * kPRing + 14);
    if (tid == 0) {
        for (int s = 0; s < kPRing; s++) { mbar_init(ringFull(s), 1); mbar_init(ringEmpty(s), 4); }
        for (int s = 0; s < 2; s++) { mbar_init(kFull(s), 4); mbar_init(kEmpty(s), 1); mbar_init(vFull(s), 4); mbar_init(vEmpty(s), 1); }
        for (int s = 0; s < 3; s++) { mbar_init(sFull(s), 1); mbar_init(pReady(s), 8); }
        mbar_init(qReady, 4);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 13) tmem_alloc(smem_u32(&s_tmem), 512);
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
        float c = 1.0f, top = -INFINITY, sum = 0.0f;
        if (tiles > 0) {
            if (part == 0) {
                s_max[0][row] = c = query_row<NB>(p, m, head, pos + t0 + token, on, smem, smem + S::kTile, row);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(qReady);
            }
            meet();
            c = s_max[0][row];
            meet();
        }
        const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
        bool ok = true;
        for (int j = 0; j < tiles; j++) {
            if (!__all_sync(0xffffffffu, mbar_wait(sFull(j % 3), (j / 3) & 1, &s_abort, p.error, 341))) ok = false;
            tc_fence_after();
            uint32_t v[64];
            const uint32_t at = mine + (uint32_t)(j % 3 * kPT + part * 64);
            tmem_ld64(at, v);
            const int left = last - j * kPT - part * 64;                 // newest key within these 64
            if (!__all_sync(0xffffffffu, left >= 63)) {
#pragma unroll
                for (int k = 0; k < 64; k++)
                    if (k > left) v[k] = 0xff800000u;
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 64; k++) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(v[k]));
            float most = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c;
            s_max[part][row] = most;
            meet();
            most = fmaxf(most, s_max[1 - part][row]);
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
                sum *= f;
                top = now;
            }
            const float shift = top > -INFINITY ? -top : 0.0f;           // a row without keys yet: every weight is 2^-inf
            float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t w[32];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float x = ex2(fmaf(__uint_as_float(v[32 * q + 2 * k]), c, shift)), y = ex2(fmaf(__uint_as_float(v[32 * q + 2 * k + 1]), c, shift));
                    s4[k & 3] += x + y;
                    split_half(x, y, w[k], w[16 + k]);
                }
                tmem_st32(at + q * 32, w);                               // 32 keys: sixteen columns hi, sixteen lo
            }
            sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pReady(j % 3));
            meet();                                                      // the maxima are read
        }
        if (tiles > 0) {
            s_max[part][row] = sum;
            meet();
            sum += s_max[1 - part][row];
        }
        if (tiles > 0 && __all_sync(0xffffffffu, ok && mbar_wait(vEmpty((tiles - 1) & 1), ((tiles - 1) >> 1) & 1, &s_abort, p.error, 343))) {
            tc_fence_after();
            const float inv = 1.0f / sum;
            float* const to = p.out + (size_t)m * p.ldo + head * HD;
#pragma unroll 1
            for (int k = 32 * part; k < HD; k += 64) {
                uint32_t o[32];
                tmem_ld32(mine + kO + k, o);
                if (on)
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(to + k + i) = make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv, __uint_as_float(o[i + 2]) * inv,
                                                                            __uint_as_float(o[i + 3]) * inv);
            }
            if (part == 0 && on && p.stats != nullptr && t0 + token >= room - p.window)
                *reinterpret_cast<float2*>(p.stats + ((size_t)m * p.H + head) * 2) = make_float2(top, sum);
        }
    } else if (warp < 12) {
        const int w = warp - 8;                   // page of the tile
        bool ok = true;
        int item = 0;
        auto convert = [&](int j, bool value) {
            const uint32_t empty = value ? vEmpty(j & 1) : kEmpty(j & 1), full = value ? vFull(j & 1) : kFull(j & 1);
            if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(empty, ((j >> 1) - 1) & 1, &s_abort, p.error, 344))) return false;
            if (!__all_sync(0xffffffffu, mbar_wait(ringFull(item % kPRing), (item / kPRing) & 1, &s_abort, p.error, 345))) return false;
            unsigned char* const tile = smem + (value ? 4 + (j & 1) : 2 + (j & 1)) * S::kTile;
            if (4 * j + w < pages) convert_row<NB>(smem + S::kRingAt + item % kPRing * S::kStage + w * Q4Page<NB>::kHalf, lane, tile, 32 * w + lane);
            else if (value) zero_row<NB>(tile, 32 * w + lane);           // weights of 0 meet no garbage
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) { mbar_arrive(ringEmpty(item % kPRing)); mbar_arrive(full); }
            item++;
            return true;
        };
        for (int j = 0; j <= tiles && ok; j++) {  // K 0, K 1, V 0, K 2, V 1, …
            if (j < tiles) ok = convert(j, false);
            if (ok && j > 0) ok = convert(j - 1, true);
        }
    } else if (warp == 12) {
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
            const uint32_t qh = base, ql = base + S::kTile;
            auto scores = [&](int j) {
                if (!mbar_wait(kFull(j & 1), (j >> 1) & 1, &s_abort, p.error, 347)) return false;
                // P·V of tile j - 3 has read this buffer
                if (j >= 3 && !mbar_wait(vEmpty((j - 3) & 1), ((j - 3) >> 1) & 1, &s_abort, p.error, 348)) return false;
                tc_fence_after();
                const uint32_t k0 = base + (2 + (j & 1)) * S::kTile, d = tmem + (uint32_t)(j % 3 * kPT);
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint32_t at = (uint32_t)((k >> 2) * (kPT * 128) + (k & 3) * 32);
                        umma_f16(d, desc_k((h ? ql : qh) + at), desc_k(k0 + at), kIdescQK, (h | k) != 0);
                    }
                umma_commit(kEmpty(j & 1));
                umma_commit(sFull(j % 3));
                return true;
            };
            bool ok = mbar_wait(qReady, 0, &s_abort, p.error, 349) && scores(0);
            for (int j = 0; j < tiles && ok; j++) {
                if (j + 1 < tiles) ok = scores(j + 1);
                if (!ok || !mbar_wait(vFull(j & 1), (j >> 1) & 1, &s_abort, p.error, 347) || !mbar_wait(pReady(j % 3), (j / 3) & 1, &s_abort, p.error, 348)) break;
                tc_fence_after();
                const uint32_t v0 = base + (4 + (j & 1)) * S::kTile, a = tmem + (uint32_t)(j % 3 * kPT);
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < kPT / 16; k++) umma_f16_ta(tmem + kO, a + (k >> 1) * 32 + h * 16 + (k & 1) * 8, desc_mn(v0 + k * 2048), kIdescPV, (j | h | k) != 0);
                umma_commit(vEmpty(j & 1));
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 13) { tc_fence_after(); tmem_dealloc(tmem, 512); }
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
            convert_row<NB>(half, lane, smem + 2 * S::kTile, tid);
        } else zero_row<NB>(smem + 2 * S::kTile, tid);
        int phase = 0;
        for (int r0 = 0; r0 < rows; r0 += kPT) {
            const int r = r0 + tid, t = room - window + r / p.ratio, head = g * p.ratio + r % p.ratio, m = first + t;
            const bool on = r < rows;
            const float c = query_row<NB>(p, m, head, pos + t, on, smem, smem + S::kTile, tid);
            float2 st = make_float2(0.0f, 1.0f);
            if (on) st = *reinterpret_cast<const float2*>(p.stats + ((size_t)m * p.H + head) * 2);
            s_row[tid] = make_float4(c, -st.x, 1.0f / st.y, __int_as_float(on ? len + t : -1));
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
