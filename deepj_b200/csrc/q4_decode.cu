// One new token per sequence over the 4-bit cache: rotation, append, attention and accumulated weights.
//
// A warp streams pages of 32 rows through a ring of its own, one bulk copy each, and keeps the running maximum and sum of the softmax in fp32.  Both
// products run on the integer tensor pipe, exactly:
//   scores   A = 16 rows × 32 dims of int8 codes (a masked page word is an operand register), B = the query in fixed point, 31 bits of its largest
//            value, as four signed base-256 digits.  A 32-dim block's integer sums are multiplied by the row's scale in fp32.
//   values   A = 16 dims × 32 rows (a byte transpose of four rows' words), B = weight × scale of the row and block, in fixed point of the page's
//            largest such product, three digits again.
// Columns 2t and 2t + 1 of B are digit t of two heads, so a lane sees one digit of up to two heads per tile and the digits meet in shuffles.  (With three digits of
// the query, which leaves two columns empty, one value of 2^12 times the others cost these all but ten bits, also where no key had anything there.)
// The new row is quantized by the warp that holds its page, into the page's copy in shared memory and into the cache: later steps read what this one did.
//
// Few heads: a cluster of up to eight blocks shares a sequence and head and exchanges maxima, sums and unnormalised rows through distributed shared
// memory.  Many: all pages of all sequences and heads in a row are dealt out evenly to the warps of a grid that fills the chip once (k_q4_stream).  A warp
// writes the output of a head whose pages it has all seen; of the first and the last one, which it may share with its neighbours, it leaves a record for
// k_q4_finish.  One block per head instead, 16 sequences of 1024 … 2048 rows and 32 heads: 46 µs with a third of the chip idle at the end.
// Weights are added up from the scores, which wait in the workspace until a row's maximum and sum are known: B · H · (rows of the cache, whatever the lengths)
// floats.
// 16 sequences of 1024 … 2048 rows and 32 heads of 128 with weights: 38.8 µs, 4.2 TB/s of the cache's bytes while the stream runs; 4 of 32700 and 32/8 heads
// 62 µs.  No unit is at its limit there (57 and 62 % of the issue slots, ALU 46 %): the latency of a page's chain of some 600 … 900 instructions, with the 16 and
// 12 warps that an SM has registers for.  Small steps are the launch and a page's latency: one sequence of 2048, 32 heads 10.2 µs.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "q4_cache.cuh"
#include "tc_common.cuh"

namespace dj {
namespace {

constexpr int kDecWarps = 4;
constexpr int kDecCluster = 8;                 // up to so many splits are a cluster
constexpr int kErrQ4Page = 334;                // device error code: a page never arrived
constexpr int kDecSpin = 1 << 22;

struct DecodeParams {
    const float* qkv; int q_off, k_off, v_off, ld;
    unsigned char* cache; int maxSeq, pages;
    const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    float* out; int ldo; int H, G, ratio, headBlocks; float scale;      // scale: 1/sqrt(hd) · log2(e)
    const float* acc; float* accOut;
    float* scores;                             // [B][H][pages · 32], log2 units; null: weights are not wanted
    float* records;                            // k_q4_stream: [2 · warps][heads of a block][hd + 2]
    float* ml;                                 // … [B][H][2] maximum and sum of a head that one warp has seen all of
    int* owners;                               // … [B][G · headBlocks][2] the warps with a head's first and last page
    int B;
    int early; int* error;
};

__device__ __forceinline__ void mma_q4(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int c) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c));
}
// the accumulator starts at the bits of 1.5 · 2^23: as a float it is that plus the integer sum, |sum| < 2^22
constexpr int kMagic = 0x4B400000;
__device__ __forceinline__ float from_magic(int v) { return __int_as_float(v) - 12582912.0f; }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float warp_max(float x) { float y; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x)); return y; }
// For |x| <= most: the power of two that brings x to fixed point below 2^22, and its inverse.  Magnitudes under 2^-100 count as nothing.
__device__ __forceinline__ float fixed_of(float most, float& back) {
    const int e = __float_as_int(fmaxf(most, 7.8886091e-31f)) & 0x7f800000;
    back = __int_as_float(e - (21 << 23));                               // 2^(e + 2 - 23)
    return __uint_as_float((275u << 23) - (uint32_t)e);
}
// x · mul in fixed point → three signed base-256 digits in the low bytes: the sum with 1.5 · 2^23 ends in the integer
__device__ __forceinline__ uint32_t digits_of(float x, float mul) { return (uint32_t)(__float_as_int(fmaf(x, mul, 12582912.0f)) + 0x408080) ^ 0x808080u; }

template <int NB> __device__ __forceinline__ void lds_piece(uint32_t (&w)[NB], const unsigned char* p) {
    if constexpr (NB == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if constexpr (NB == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}
// the NB bf16 scales of a row
template <int NB> __device__ __forceinline__ void lds_scales(float (&s)[NB], const unsigned char* p) {
    if constexpr (NB == 1) s[0] = __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(p) << 16);
    else {
        uint32_t w[NB / 2];
        if constexpr (NB == 4) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
        else w[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int i = 0; i < NB / 2; i++) { s[2 * i] = __uint_as_float(w[i] << 16); s[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
}

template <int NB, int HPB> struct DecodeShape {
    static constexpr int HD = 32 * NB, NT = (HPB + 1) / 2, CH = HPB == 1 ? 1 : 2;      // tiles of heads, heads of a tile
    static constexpr int kStages = NB == 4 ? 2 : NB == 2 ? 3 : 6;
    static constexpr int kRing = kStages * Q4Page<NB>::kBytes;           // of a warp
    static constexpr int kDigits = NB * HPB * 96;                        // … [block][head][digit][32 rows]
    static constexpr int kQuery = HPB * 4 * HD;                          // … the queries' digits
    static constexpr int kWarp = kRing + kDigits + kQuery;
    static constexpr size_t kSmem = kDecWarps * kWarp + 64;              // 64: zeros for the columns without a head
    // blocks of an SM: the stream's registers want room (16 sequences of 32 heads of 128: 37 µs with four, 41 with five); blocks that are many and short want
    // places (64 sequences of 12 heads of 64, back to back on one input: 14.4 with four, 12.3 with five, 10.3 with six), unless that spills (32 of 16 heads of
    // 128: 10.3 and, with five, 12.3)
    static constexpr int kResident = HPB == 4 ? 3 : 4, kShort = HPB == 1 && NB < 4 ? 6 : kResident;
};

// What a warp knows of the pages it is at, and its part of a sequence and head.
template <int NB, int HPB>
struct DecodeWarp {
    using S = DecodeShape<NB, HPB>;
    using Page = Q4Page<NB>;
    static constexpr int HD = S::HD, NT = S::NT, CH = S::CH, kStages = S::kStages, LPR = 8 * NB;      // LPR: lanes of a row of four values each
    const DecodeParams& p;
    unsigned char* ring; unsigned char* digits; uint32_t* query; const unsigned char* zeros;
    uint32_t bars;
    int lane, g, t, e, asked = 0, taken = 0, limit = kDecSpin;
    float m[HPB], l[HPB], factor[NT][CH], acc[NT][NB][2][2 * CH];        // acc: [tile of heads][block][half][row g, row g + 8 × heads]
    uint32_t bq[NT][NB][2];

    __device__ __forceinline__ DecodeWarp(const DecodeParams& params, unsigned char* smem, unsigned long long* bar, int warp) : p(params) {
        ring = smem + warp * S::kWarp;
        digits = ring + S::kRing;
        query = reinterpret_cast<uint32_t*>(digits + S::kDigits);
        zeros = smem + kDecWarps * S::kWarp;
        lane = threadIdx.x & 31; g = lane >> 2; t = lane & 3; e = lane % LPR;
        bars = smem_u32(bar + warp * kStages);
        if (lane < kStages) mbar_init(bars + 8 * lane, 1);
        if (threadIdx.x < 16) reinterpret_cast<uint32_t*>(smem + kDecWarps * S::kWarp)[threadIdx.x] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void restart() {                          // every page asked for has been taken: the barriers' phases begin anew
        asked = taken = 0;
        if (lane < kStages) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bars + 8 * lane) : "memory"); mbar_init(bars + 8 * lane, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void request(const unsigned char* page) {
        if (lane == 0) {
            const uint32_t bar = bars + 8 * (asked % kStages);
            mbar_arrive_expect_tx(bar, Page::kBytes);
            bulk_g2s(smem_u32(ring + asked % kStages * Page::kBytes), page, Page::kBytes, bar);
        }
        asked++;
    }
    __device__ __forceinline__ unsigned char* take() {
        const uint32_t bar = bars + 8 * (taken % kStages), parity = (taken / kStages) & 1;
        bool ready = mbar_try_wait(bar, parity);
#pragma unroll 1
        for (int spin = 0; !ready && spin < limit; spin++) ready = mbar_try_wait(bar, parity);
        if (!ready) {                             // never on a healthy device: flag it, stop waiting long, keep the control flow
            if (lane == 0) atomicCAS(p.error, 0, kErrQ4Page);
            limit = 64;
        }
        return ring + taken++ % kStages * Page::kBytes;
    }

    // A head's query, rotated, in fixed point of its largest value → its digits at `to`; returns the factor of its sums, in log2 units.
    __device__ __forceinline__ float put_query(uint32_t* to, float4 q, const float2& cs, const float2& sn) const {
        q = q4_rotate(q, cs, sn);
        float back, bad = fmaf(q.x, 0.0f, fmaf(q.y, 0.0f, fmaf(q.z, 0.0f, q.w * 0.0f)));
        const float mul = fixed_of(warp_max(fmaxf(fmaxf(fabsf(q.x), fabsf(q.y)), fmaxf(fabsf(q.z), fabsf(q.w)))), back);
        bad = __any_sync(0xffffffffu, bad != bad) ? __int_as_float(0x7fc00000) : 0.0f;      // NaN where the query holds an infinity or a NaN
        auto digits4 = [&](float x) { return ((uint32_t)__float2int_rn(x * mul * 256.0f) + 0x808080u) ^ 0x808080u; };      // below 2^30
        const uint32_t u0 = digits4(q.x), u1 = digits4(q.y), u2 = digits4(q.z), u3 = digits4(q.w);
        const uint32_t t0 = __byte_perm(u0, u1, 0x5140), t1 = __byte_perm(u2, u3, 0x5140), t2 = __byte_perm(u0, u1, 0x7362), t3 = __byte_perm(u2, u3, 0x7362);
        if (lane < LPR) {
            to[3 * (HD / 4) + e] = __byte_perm(t0, t1, 0x5410);
            to[2 * (HD / 4) + e] = __byte_perm(t0, t1, 0x7632);
            to[HD / 4 + e] = __byte_perm(t2, t3, 0x5410);
            to[e] = __byte_perm(t2, t3, 0x7632);
        }
        return back * p.scale * (1.0f / 16.0f) + bad;
    }
    __device__ __forceinline__ float digit() const { return t == 0 ? 65536.0f : t == 1 ? 256.0f : t == 2 ? 1.0f : 0.0f; }      // what this lane's digit of a weight counts for
    __device__ __forceinline__ float query_digit() const { return t == 3 ? 1.0f / 256.0f : digit(); }
    // Operands from all heads' digits; an empty softmax.
    __device__ __forceinline__ void begin(const uint32_t* queries, const float* factors) {
        const int hc = g & 1, dc = g >> 1;        // head and digit of the B column this lane fills
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const bool on = 2 * n + hc < HPB;
            const uint32_t* const from = queries + (on ? ((2 * n + hc) * 4 + dc) * (HD / 4) : 0);
#pragma unroll
            for (int j = 0; j < NB; j++) {
                bq[n][j][0] = on ? from[8 * j + t] : 0;
                bq[n][j][1] = on ? from[8 * j + 4 + t] : 0;
            }
#pragma unroll
            for (int c = 0; c < CH; c++) factor[n][c] = factors[2 * n + c] * query_digit();
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int k = 0; k < 2 * CH; k++) acc[n][j][x][k] = 0.0f;
        }
#pragma unroll
        for (int h = 0; h < HPB; h++) { m[h] = -INFINITY; l[h] = 0.0f; }
    }

    // The new row's key and value → row r of the page in shared memory and, by one of the head blocks, in the cache.
    __device__ __forceinline__ void put_row(const float* row, int head, const float2& cs, const float2& sn, unsigned char* page, unsigned char* cached, int r) const {
        const float4 kx = q4_rotate(*reinterpret_cast<const float4*>(row + p.k_off + head * HD + 4 * e), cs, sn);
        const float4 vx = *reinterpret_cast<const float4*>(row + p.v_off + head * HD + 4 * e);
        q4_put_row<NB>(page, r, false, e, kx, lane < LPR);
        q4_put_row<NB>(page, r, true, e, vx, lane < LPR);
        if (cached != nullptr) {
            q4_put_row<NB>(cached, r, false, e, kx, lane < LPR);
            q4_put_row<NB>(cached, r, true, e, vx, lane < LPR);
        }
        __syncwarp();
    }

    // One page of `left` rows.  waiting: where head 0's scores of this page go (the next head's `pitch` floats on), or null.
    __device__ __forceinline__ void step(const unsigned char* page, int left, float* waiting, size_t pitch, int heads) {
        const int key = 8 * t + g;                // the row that this lane's weights are of
        // byte (row / 4 % 4) of word (row % 4, row / 16) of an operand
        unsigned char* const put = digits + (key & 3) * 8 + (key >> 4) * 4 + ((key >> 2) & 3);
        const uint32_t pick = g & 1 ? 0x7362u : 0x5140u;
        // scores: rows 8k + g in s[n][head][k]
        float s[NT][CH][4];
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            uint32_t wa[NB], wb[NB];
            float sa[NB], sb[NB];
            lds_piece<NB>(wa, page + Page::word(16 * mt + g, t, 0));
            lds_piece<NB>(wb, page + Page::word(16 * mt + 8 + g, t, 0));
            lds_scales<NB>(sa, page + Page::kKs + (16 * mt + g) * NB * 2);
            lds_scales<NB>(sb, page + Page::kKs + (16 * mt + 8 + g) * NB * 2);
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const uint32_t a[4] = {q4_low(wa[j]), q4_low(wb[j]), q4_high(wa[j]), q4_high(wb[j])};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    int d[4];
                    mma_q4(d, a, bq[n][j][0], bq[n][j][1], kMagic);
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        s[n][c][2 * mt] = j == 0 ? from_magic(d[c]) * sa[0] : fmaf(from_magic(d[c]), sa[j], s[n][c][2 * mt]);
                        s[n][c][2 * mt + 1] = j == 0 ? from_magic(d[2 + c]) * sb[0] : fmaf(from_magic(d[2 + c]), sb[j], s[n][c][2 * mt + 1]);
                    }
                }
            }
        }
        const bool in = key < left;
        float vs[NB], back[HPB][NB];
        lds_scales<NB>(vs, page + Page::kVs + key * NB * 2);
#pragma unroll
        for (int h = 0; h < HPB; h++) {
            // the digits meet, and every lane gets its row's sum: two exchanges of halves
            const float f = factor[h / 2][h % 2], s0 = s[h / 2][h % 2][0] * f, s1 = s[h / 2][h % 2][1] * f, s2 = s[h / 2][h % 2][2] * f, s3 = s[h / 2][h % 2][3] * f;
            const float a = (t & 1 ? s1 : s0) + __shfl_xor_sync(0xffffffffu, t & 1 ? s0 : s1, 1), b = (t & 1 ? s3 : s2) + __shfl_xor_sync(0xffffffffu, t & 1 ? s2 : s3, 1);
            float sc = (t & 2 ? b : a) + __shfl_xor_sync(0xffffffffu, t & 2 ? a : b, 2);
            if (waiting != nullptr && h < heads) waiting[h * pitch + key] = sc;
            sc = in ? sc : -INFINITY;
            const float now = fmaxf(m[h], warp_max(sc));
            if (now > m[h]) {                     // seldom after the first pages
                const float fall = ex2(m[h] - now);
                l[h] *= fall;
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int x = 0; x < 2; x++) { acc[h / 2][j][x][h % 2] *= fall; acc[h / 2][j][x][CH + h % 2] *= fall; }
                m[h] = now;
            }
            const float w = in ? ex2(sc - m[h]) : 0.0f;
            l[h] += w;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const float x = w * vs[j];
                const uint32_t u = digits_of(x, fixed_of(warp_max(x), back[h][j]));
                unsigned char* const to = put + (j * HPB + h) * 96;
                to[0] = (unsigned char)(u >> 16); to[32] = (unsigned char)(u >> 8); to[64] = (unsigned char)u;
            }
        }
        __syncwarp();
        // values
        const int hc = g & 1, dc = g >> 1;
        uint32_t v[8][NB];
#pragma unroll
        for (int i = 0; i < 8; i++) lds_piece<NB>(v[i], page + Page::kV + Page::word(16 * (i >> 2) + t + 4 * (i & 3), g >> 1, 0));
#pragma unroll
        for (int j = 0; j < NB; j++) {
            uint32_t lo[2], hi[2];                // bytes of the even and the odd dim of four rows, low and high nibble 16 dims apart
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t x01 = __byte_perm(v[4 * k][j], v[4 * k + 1][j], pick), x23 = __byte_perm(v[4 * k + 2][j], v[4 * k + 3][j], pick);
                lo[k] = __byte_perm(x01, x23, 0x5410);
                hi[k] = __byte_perm(x01, x23, 0x7632);
            }
            const uint32_t a0[4] = {q4_low(lo[0]), q4_low(hi[0]), q4_low(lo[1]), q4_low(hi[1])};
            const uint32_t a1[4] = {q4_high(lo[0]), q4_high(hi[0]), q4_high(lo[1]), q4_high(hi[1])};
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const bool on = dc < 3 && 2 * n + hc < HPB;
                const uint2 bw = *reinterpret_cast<const uint2*>(on ? digits + (j * HPB + 2 * n + hc) * 96 + dc * 32 + t * 8 : zeros);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    int d[4];
                    mma_q4(d, x ? a1 : a0, bw.x, bw.y, kMagic);
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        acc[n][j][x][c] = fmaf(from_magic(d[c]), back[2 * n + c][j], acc[n][j][x][c]);
                        acc[n][j][x][CH + c] = fmaf(from_magic(d[2 + c]), back[2 * n + c][j], acc[n][j][x][CH + c]);
                    }
                }
            }
        }
        fence_proxy_async_smem();                 // the next copy comes over the page
        __syncwarp();                             // the page and the digits are read out
    }

    // Sums over the warp: l, and the unnormalised row of head h with its digits added up, times `scale`; lanes t < 2 hand two halves of 16 values to `out`.
    template <typename Out>
    __device__ __forceinline__ void row(int h, float scale, Out out) const {
        const float f = digit() * (1.0f / 16.0f) * scale;
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const float a = acc[h / 2][j][x][h % 2] * f, b = acc[h / 2][j][x][CH + h % 2] * f;
                float v = (t & 1 ? b : a) + __shfl_xor_sync(0xffffffffu, t & 1 ? a : b, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (t < 2) out(32 * j + 16 * x + 2 * g + t, v);
            }
    }
    __device__ __forceinline__ void sums() {
#pragma unroll
        for (int h = 0; h < HPB; h++)
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    }
};

__device__ __forceinline__ float weight_of(float mine, float top) { return mine > -INFINITY ? ex2(mine - top) : 0.0f; }

// ───────────── few heads: clusters ─────────────
// grid (splits, heads of the cache × blocks of query heads, sequences); warps take a split's pages in turn.
template <int NB, int HPB, bool CLUSTER>
__global__ void __launch_bounds__(kDecWarps * 32, DecodeShape<NB, HPB>::kShort) k_q4_decode(const DecodeParams p) {
    using S = DecodeShape<NB, HPB>;
    using Page = Q4Page<NB>;
    constexpr int HD = S::HD, kOut = HPB * HD, W = kDecWarps;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) unsigned long long s_bar[W * S::kStages];
    __shared__ __align__(16) uint32_t s_q[HPB * 4 * HD / 4];
    __shared__ float s_factor[HPB], s_m[W][HPB], s_l[W][HPB], s_own[HPB][2];
    __shared__ float s_ml[CLUSTER ? kDecCluster : 1][HPB][2];            // every split's maximum and sum
    __shared__ float s_red[CLUSTER ? kOut : 1];                          // this block's share of the output row, of every split
    const int split = blockIdx.x, splits = gridDim.x, head = blockIdx.y / p.headBlocks, hb = blockIdx.y - head * p.headBlocks, b = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5;
    const int heads = min(HPB, p.ratio - hb * HPB), h0 = head * p.ratio + hb * HPB;
    if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    DecodeWarp<NB, HPB> w(p, smem, s_bar, warp);
    unsigned char* const plane = p.cache + ((size_t)b * p.G + head) * p.pages * Page::kBytes;
    int len = 0, pos = 0, first = 0, end = 0;
    bool there = false;
    auto place = [&]() {                          // where this sequence stands
        len = q4_int(__ldcg(p.len + b)); pos = q4_int(__ldcg(p.pos + b));
        there = q4_room(1, len, p.maxSeq, pos, p.maxPos) == 1;
        const int pages = len / kQ4Page + 1, share = (pages + splits - 1) / splits;
        first = min(pages, split * share);
        end = there ? min(pages, first + share) : first;
    };
    auto request = [&]() {
        const int pg = first + warp + w.asked * W;
        if (pg < end) w.request(plane + (size_t)pg * Page::kBytes);
    };
    // Behind a projection of the same stream the cached rows are complete: the first pages are asked for before the dependency wait.  A length that
    // has moved by then (never observed) drops them.
    int before = -1;
    if (p.early) {
        place();
        before = there ? len : -1;
#pragma unroll 1
        for (int i = 0; i < S::kStages; i++) request();
    }
    pdl_wait();
    pdl_launch_dependents();
    const float* const row = p.qkv + (size_t)b * p.ld;
    float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (warp < heads) q = *reinterpret_cast<const float4*>(row + p.q_off + (h0 + warp) * HD + 4 * w.e);
    place();
    if (before >= 0 && (!there || len != before)) {
#pragma unroll 1
        while (w.taken < w.asked) w.take();
        __syncwarp();
        w.restart();
        before = -1;
    }
    if (!there) {                                 // the whole cluster: it shares the sequence
        if constexpr (CLUSTER) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    if (before < 0)
#pragma unroll 1
        for (int i = 0; i < S::kStages; i++) request();
    const size_t tab = (size_t)pos * (HD / 2) + 2 * w.e;
    const float2 cs = *reinterpret_cast<const float2*>(p.cosT + tab), sn = *reinterpret_cast<const float2*>(p.sinT + tab);
    if (warp < HPB) {
        const float f = w.put_query(s_q + warp * 4 * (HD / 4), q, cs, sn);
        if (w.lane == 0) s_factor[warp] = f;
    }
    __syncthreads();
    w.begin(s_q, s_factor);
    const size_t pitch = (size_t)p.pages * kQ4Page;
    float* const waiting = p.scores == nullptr ? nullptr : p.scores + ((size_t)b * p.H + h0) * pitch;
#pragma unroll 1
    for (int pg = first + warp; pg < end; pg += W) {
        unsigned char* const page = w.take();
        if (pg == len / kQ4Page) w.put_row(row, head, cs, sn, page, hb == 0 ? plane + (size_t)pg * Page::kBytes : nullptr, len % kQ4Page);
        w.step(page, len + 1 - pg * kQ4Page, waiting == nullptr ? nullptr : waiting + pg * kQ4Page, pitch, heads);
        request();
    }

    // the warps' rows meet in the rings' memory, where nothing is on its way any more
    __syncthreads();
    float* const part = reinterpret_cast<float*>(smem);                  // [warp][head][HD]
    w.sums();
#pragma unroll
    for (int h = 0; h < HPB; h++) {
        if (w.lane == 0) { s_m[warp][h] = w.m[h]; s_l[warp][h] = w.l[h]; }
        w.row(h, 1.0f, [&](int d, float v) { part[(warp * HPB + h) * HD + d] = v; });
    }
    __syncthreads();
    if (tid < HPB) {                              // the block's maximum and sum, and what every warp's row counts for
        float top = -INFINITY, sum = 0.0f;
        for (int i = 0; i < W; i++) top = fmaxf(top, s_m[i][tid]);
        for (int i = 0; i < W; i++) {
            const float f = weight_of(s_m[i][tid], top);
            sum = fmaf(s_l[i][tid], f, sum);
            s_m[i][tid] = f;
        }
        s_own[tid][0] = top; s_own[tid][1] = sum;
    }
    __syncthreads();
    auto block_row = [&](int i) {
        float a = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) a = fmaf(part[k * kOut + i], s_m[k][i / HD], a);
        return a;
    };
    float* const orow = p.out + (size_t)b * p.ldo + h0 * HD;
    if (!CLUSTER) {
        for (int i = tid; i < heads * HD; i += W * 32) orow[i] = block_row(i) / s_own[i / HD][1];
    } else {
        __syncwarp();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // every block of the cluster is running
        const int share = kOut / splits;          // elements of the row that a block adds up
        auto put_to = [](const float* at, int rank, float x) {
            uint32_t a;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(at)), "r"(rank));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory");
        };
        for (int i = tid; i < kOut; i += W * 32) put_to(&s_red[split * share + i % share], i / share, block_row(i));
        if (tid < HPB * splits) { put_to(&s_ml[split][tid % HPB][0], tid / HPB, s_own[tid % HPB][0]); put_to(&s_ml[split][tid % HPB][1], tid / HPB, s_own[tid % HPB][1]); }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = tid; i < share; i += W * 32) {
            const int at = split * share + i, h = at / HD;
            float top = -INFINITY, sum = 0.0f, a = 0.0f;
            for (int r = 0; r < splits; r++) top = fmaxf(top, s_ml[r][h][0]);
            for (int r = 0; r < splits; r++) {
                const float f = weight_of(s_ml[r][h][0], top);
                sum = fmaf(s_ml[r][h][1], f, sum);
                a = fmaf(s_red[r * share + i], f, a);
            }
            if (h < heads) orow[at] = a / sum;
        }
    }
    if (waiting == nullptr) return;
    // this block's rows: their old weights and those of this step
    float top[HPB], inv[HPB];
#pragma unroll
    for (int h = 0; h < HPB; h++) {
        top[h] = CLUSTER ? -INFINITY : s_own[h][0];
        float sum = CLUSTER ? 0.0f : s_own[h][1];
        if constexpr (CLUSTER) {
            for (int r = 0; r < splits; r++) top[h] = fmaxf(top[h], s_ml[r][h][0]);
            for (int r = 0; r < splits; r++) sum = fmaf(s_ml[r][h][1], weight_of(s_ml[r][h][0], top[h]), sum);
        }
        inv[h] = 1.0f / sum;
    }
    const size_t at = ((size_t)b * p.G + head) * p.maxSeq;
    const int last = min(len + 1, end * kQ4Page);
#pragma unroll 1
    for (int i0 = first * kQ4Page + tid; i0 < last; i0 += 4 * W * 32) {  // four rows a time: the loads' latency is most of it
        float add[4], old[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * W * 32;
            old[k] = i < min(last, len) ? p.acc[at + i] : 0.0f;
            add[k] = 0.0f;
#pragma unroll
            for (int h = 0; h < HPB; h++)
                if (i < last && h < heads) add[k] = fmaf(ex2(waiting[h * pitch + i] - top[h]), inv[h], add[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i0 + k * W * 32 < last) p.accOut[at + i0 + k * W * 32] = old[k] + add[k];
    }
}

// ───────────── many heads: all pages in a row ─────────────
// The row: for every sequence, for every head of the cache and block of query heads, kHeadUnits for what a warp does before the first and after the last
// page, and its pages.  Warp i of N has units U·i/N … U·(i + 1)/N of U.  (Counted by pages alone, the warps that got the heads of a sequence of one
// page took twice as long as all others.)
constexpr int kHeadUnits = 4;
__device__ __forceinline__ int pages_of(const DecodeParams& p, int b, int& len, int& pos) {
    len = q4_int(p.len[b]); pos = q4_int(p.pos[b]);
    return q4_room(1, len, p.maxSeq, pos, p.maxPos) == 1 ? len / kQ4Page + 1 : 0;
}
__device__ __forceinline__ long long units_of(int pages, int heads) { return pages > 0 ? (long long)(pages + kHeadUnits) * heads : 0; }
struct StreamPlace {
    int b, seg, pages, len, pos;                  // the sequence, its head, its pages
    int page, end;                                // this warp's pages of it that are left; none: the warp is through
    long long units;                              // units of the warp behind this head
    __device__ __forceinline__ void enter(int off) {
        const int upto = (int)min((long long)pages + kHeadUnits, off + units);
        page = max(0, off - kHeadUnits);
        end = max(0, upto - kHeadUnits);
        units -= upto - off;
    }
    __device__ __forceinline__ void next(const DecodeParams& p) {
        page = end = 0;
        while (units > 0 && page >= end) {
            if (++seg == p.G * p.headBlocks) {
                seg = 0;
                do pages = pages_of(p, ++b, len, pos); while (pages == 0);
            }
            enter(0);
        }
    }
};

template <int NB, int HPB>
__global__ void __launch_bounds__(kDecWarps * 32, DecodeShape<NB, HPB>::kResident) k_q4_stream(const DecodeParams p) {
    using S = DecodeShape<NB, HPB>;
    using Page = Q4Page<NB>;
    constexpr int HD = S::HD;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) unsigned long long s_bar[kDecWarps * S::kStages];
    __shared__ float s_factor[kDecWarps][HPB];
    __shared__ StreamPlace s_at[kDecWarps], s_ask[kDecWarps];            // out of the way of the loop's registers
    const int warp = threadIdx.x >> 5, heads_ = p.G * p.headBlocks;
    DecodeWarp<NB, HPB> w(p, smem, s_bar, warp);
    const int lane = w.lane;
    __syncthreads();                              // the zeros stand
    pdl_wait();
    pdl_launch_dependents();
    long long total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        int len, pos;
        long long n = b0 + lane < p.B ? units_of(pages_of(p, b0 + lane, len, pos), heads_) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        total += n;
    }
    const int me = blockIdx.x * kDecWarps + warp, all = (int)min((long long)gridDim.x * kDecWarps, total);
    const long long from = me < all ? total * me / all : total;
    const long long upTo = me < all ? total * (me + 1) / all : total;
    if (from >= upTo) return;
    const unsigned char* askPage = nullptr;       // the next page to ask for, and how many of its head are left
    int askLeft;
    {
        StreamPlace at = {};
        at.units = upTo - from;
        long long base = 0;
        bool found = false;
        for (int b0 = 0; b0 < p.B && !found; b0 += 32) {
            int len = 0, pos = 0;
            const int pages = b0 + lane < p.B ? pages_of(p, b0 + lane, len, pos) : 0;
            const long long n = units_of(pages, heads_);
            long long upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const long long v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
            const unsigned hit = __ballot_sync(0xffffffffu, from < base + upto);
            if (hit) {
                const int k = __ffs(hit) - 1;
                const long long off = from - base - __shfl_sync(0xffffffffu, upto - n, k);
                at.b = b0 + k;
                at.pages = __shfl_sync(0xffffffffu, pages, k); at.len = __shfl_sync(0xffffffffu, len, k); at.pos = __shfl_sync(0xffffffffu, pos, k);
                at.seg = (int)(off / (at.pages + kHeadUnits));
                at.enter((int)(off - (long long)at.seg * (at.pages + kHeadUnits)));
                if (at.page >= at.end) at.next(p);
                found = true;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) s_at[warp] = s_ask[warp] = at;
        __syncwarp();
        askLeft = at.end - at.page;
        askPage = p.cache + (((size_t)at.b * p.G + at.seg / p.headBlocks) * p.pages + at.page) * Page::kBytes;
    }
    auto request = [&]() {
        if (askLeft <= 0) return;
        w.request(askPage);
        askPage += Page::kBytes;
        if (--askLeft == 0) {
            StreamPlace ask = s_ask[warp];
            ask.next(p);
            __syncwarp();
            if (lane == 0) s_ask[warp] = ask;
            __syncwarp();
            askLeft = ask.end - ask.page;
            askPage = p.cache + (((size_t)ask.b * p.G + ask.seg / p.headBlocks) * p.pages + ask.page) * Page::kBytes;
        }
    };
#pragma unroll 1
    for (int i = 0; i < S::kStages; i++) request();
    const size_t pitch = (size_t)p.pages * kQ4Page;
#pragma unroll 1
    while (true) {
        const StreamPlace& at = s_at[warp];
        const int end = at.end, len = at.len;
        if (at.page >= end) return;
        const int head = at.seg / p.headBlocks, hb = at.seg - head * p.headBlocks, heads = min(HPB, p.ratio - hb * HPB), h0 = head * p.ratio + hb * HPB;
        const float* const row = p.qkv + (size_t)at.b * p.ld;
        const size_t tab = (size_t)at.pos * (HD / 2) + 2 * w.e;
        const float2 cs = *reinterpret_cast<const float2*>(p.cosT + tab), sn = *reinterpret_cast<const float2*>(p.sinT + tab);
        float4 q[HPB];
#pragma unroll
        for (int h = 0; h < HPB; h++) q[h] = h < heads ? *reinterpret_cast<const float4*>(row + p.q_off + (h0 + h) * HD + 4 * w.e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int h = 0; h < HPB; h++) {
            const float f = w.put_query(w.query + h * 4 * (HD / 4), q[h], cs, sn);
            if (lane == 0) s_factor[warp][h] = f;
        }
        __syncwarp();
        w.begin(w.query, s_factor[warp]);
        float* const waiting = p.scores == nullptr ? nullptr : p.scores + ((size_t)at.b * p.H + h0) * pitch;
        unsigned char* const plane = p.cache + ((size_t)at.b * p.G + head) * p.pages * Page::kBytes;
#pragma unroll 1
        for (int pg = at.page; pg < end; pg++) {
            unsigned char* const page = w.take();
            if (pg == len / kQ4Page) w.put_row(p.qkv + (size_t)at.b * p.ld, head, cs, sn, page, hb == 0 ? plane + (size_t)pg * Page::kBytes : nullptr, len % kQ4Page);
            w.step(page, len + 1 - pg * kQ4Page, waiting == nullptr ? nullptr : waiting + pg * kQ4Page, pitch, heads);
            request();
        }
        w.sums();
        const bool whole = at.page == 0 && at.end == at.pages;
        float* const record = p.records + (size_t)(2 * me + (at.page > 0 ? 0 : 1)) * HPB * (HD + 2);
#pragma unroll
        for (int h = 0; h < HPB; h++)
            if (h < heads) {
                float* const to = whole ? p.out + (size_t)at.b * p.ldo + (h0 + h) * HD : record + h * (HD + 2);
                w.row(h, whole ? 1.0f / w.l[h] : 1.0f, [&](int d, float v) { to[d] = v; });
                if (lane == 0) {
                    float* const ml = whole ? p.ml + ((size_t)at.b * p.H + h0 + h) * 2 : record + h * (HD + 2) + HD;
                    ml[0] = w.m[h]; ml[1] = w.l[h];
                }
            }
        if (lane == 0) {
            int* const owners = p.owners + ((size_t)at.b * heads_ + at.seg) * 2;
            if (at.page == 0) owners[0] = me;
            if (at.end == at.pages) owners[1] = me;
        }
        StreamPlace now = at;
        now.next(p);
        __syncwarp();                             // the place and the queries' digits are read out
        if (lane == 0) s_at[warp] = now;
        __syncwarp();
    }
}

// What k_q4_stream left.  Blocks r < ratio merge the records of head r of a group, where several warps had it; the others add up the weights of 1024 rows
// of one sequence and head of the cache.
struct FinishParams {
    const float* len; const float* pos; int maxSeq, maxPos, pages;
    const float* records; const float* ml; const int* owners;
    const float* scores; const float* acc; float* accOut;
    float* out; int ldo; int H, G, ratio, headBlocks, perBlock, hd;
};
constexpr int kFinishRows = 1024;
__global__ void __launch_bounds__(256) k_q4_finish(const FinishParams p) {
    __shared__ float s_top[64], s_inv[64];
    __shared__ float4 s_sum[8][32];
    pdl_wait();
    pdl_launch_dependents();
    const int g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, len = q4_int(p.len[b]), pos = q4_int(p.pos[b]);
    if (q4_room(1, len, p.maxSeq, pos, p.maxPos) != 1) return;
    const bool merges = (int)blockIdx.x < p.ratio;
    const int from = merges ? 0 : ((int)blockIdx.x - p.ratio) * kFinishRows, rec = p.hd + 2;
    if (from > len) return;
    const size_t at = ((size_t)b * p.G + g) * p.maxSeq, pitch = (size_t)p.pages * kQ4Page;
    const float* const sc = p.scores + ((size_t)b * p.H + g * p.ratio) * pitch;
    float add[kFinishRows / 256], old[kFinishRows / 256], next[kFinishRows / 256];
    auto load = [&](int r) {                      // a head's scores, ahead of their use
#pragma unroll
        for (int k = 0; k < kFinishRows / 256; k++) next[k] = r < p.ratio && from + tid + 256 * k <= len ? sc[r * pitch + from + tid + 256 * k] : 0.0f;
    };
    if (!merges) {
#pragma unroll
        for (int k = 0; k < kFinishRows / 256; k++) { old[k] = from + tid + 256 * k < len ? p.acc[at + from + tid + 256 * k] : 0.0f; add[k] = 0.0f; }
        load(0);
    }
    // maximum and sum of head r, a warp each (in blocks that merge: the block's head)
    for (int r = merges ? (int)blockIdx.x : warp; r < p.ratio; r += 8) {
        const int hb = r / p.perBlock, h = r - hb * p.perBlock;
        const int* const own = p.owners + ((size_t)b * p.G * p.headBlocks + g * p.headBlocks + hb) * 2;
        const int i0 = own[0], n = own[1] - i0 + 1;
        auto record = [&](int i) { return p.records + ((size_t)(2 * (i0 + i) + (i == 0 ? 1 : 0)) * p.perBlock + h) * rec; };
        if (merges && n == 1) return;             // the warp that had it all has written it
        float top, sum;
        if (n == 1) {
            const float* const ml = p.ml + ((size_t)b * p.H + g * p.ratio + r) * 2;
            top = ml[0]; sum = ml[1];
        } else {
            float m0 = -INFINITY, l0 = 0.0f;      // records lane, lane + 32, …
            for (int i = lane; i < n; i += 32) {
                const float2 ml = *reinterpret_cast<const float2*>(record(i) + p.hd);
                const float now = fmaxf(m0, ml.x);
                l0 = fmaf(l0, weight_of(m0, now), ml.y * weight_of(ml.x, now));
                m0 = now;
            }
            top = warp_max(m0);
            sum = l0 * weight_of(m0, top);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (!merges) {
            if (lane == 0) { s_top[r] = top; s_inv[r] = 1.0f / sum; }
            continue;
        }
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);                  // every eighth record
        if (4 * lane < p.hd)
#pragma unroll 4
            for (int i = warp; i < n; i += 8) {
                const float* const from = record(i);
                const float2 x = *reinterpret_cast<const float2*>(from + 4 * lane), y = *reinterpret_cast<const float2*>(from + 4 * lane + 2);
                const float f = weight_of(from[p.hd], top);
                a = make_float4(fmaf(x.x, f, a.x), fmaf(x.y, f, a.y), fmaf(y.x, f, a.z), fmaf(y.y, f, a.w));
            }
        s_sum[warp][lane] = a;
        __syncthreads();
        if (warp == 0 && 4 * lane < p.hd) {
#pragma unroll
            for (int i = 1; i < 8; i++) { const float4 v = s_sum[i][lane]; a = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w); }
            *reinterpret_cast<float4*>(p.out + (size_t)b * p.ldo + (g * p.ratio + r) * p.hd + 4 * lane) = make_float4(a.x / sum, a.y / sum, a.z / sum, a.w / sum);
        }
        return;
    }
    __syncthreads();
    for (int r = 0; r < p.ratio; r++) {
        float now[kFinishRows / 256];
#pragma unroll
        for (int k = 0; k < kFinishRows / 256; k++) now[k] = next[k];
        load(r + 1);
#pragma unroll
        for (int k = 0; k < kFinishRows / 256; k++) add[k] = fmaf(ex2(now[k] - s_top[r]), s_inv[r], add[k]);
    }
#pragma unroll
    for (int k = 0; k < kFinishRows / 256; k++)
        if (from + tid + 256 * k <= len) p.accOut[at + from + tid + 256 * k] = old[k] + add[k];
}

int heads_per_block(int ratio) { return ratio >= 3 ? 4 : ratio; }

struct DecodePlan { int headBlocks, perBlock, pages, splits, blocks; bool stream; size_t scores, records, ml, owners; };
DecodePlan decode_plan(const Q4AttnArgs& a) {
    DecodePlan d = {};
    const int ratio = a.H / a.G;
    d.perBlock = heads_per_block(ratio);
    d.headBlocks = (ratio + d.perBlock - 1) / d.perBlock;
    d.pages = (a.maxSeq + kQ4Page - 1) / kQ4Page;
    d.blocks = (d.perBlock == 4 ? 3 : 4) * g_num_sms;                    // all that are resident at once
    const long long heads = (long long)a.B * a.G * d.headBlocks;
    // Clusters of up to eight where they fit onto the chip together, until a warp has a page (16 heads of 10 pages: 5.5 µs with two blocks to a head, 4.8 with
    // four).  Pages in a row where a block would have more than 32 of a head (16 sequences of 32 heads with 65 each 46 µs a block each, 41 in a row; 64 of 12
    // heads with 7 each 15 and 18.5).
    d.splits = 1;
    while (d.splits < kDecCluster && d.splits * kDecWarps < d.pages && heads * d.splits * 2 <= d.blocks) d.splits *= 2;
    d.stream = d.pages > 8 * kDecWarps * d.splits || (a.accOut != nullptr && d.headBlocks > 1);
    d.scores = a.accOut != nullptr ? (size_t)a.B * a.H * d.pages * kQ4Page : 0;
    if (d.stream) {
        d.records = (size_t)2 * d.blocks * kDecWarps * d.perBlock * (a.hd + 2);
        d.ml = (size_t)a.B * a.H * 2;
        d.owners = (size_t)heads * 2;
    }
    return d;
}

template <int NB, int HPB>
void decode(const DecodeParams& p, const DecodePlan& d, cudaStream_t s) {
    using S = DecodeShape<NB, HPB>;
    static bool attr = false;
    if (!attr) {
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_decode<NB, HPB, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_decode<NB, HPB, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_stream<NB, HPB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        attr = true;
    }
    if (d.stream) launch_k(k_q4_stream<NB, HPB>, dim3(d.blocks), dim3(kDecWarps * 32), S::kSmem, s, true, p);
    else launch_k_cluster(d.splits > 1 ? k_q4_decode<NB, HPB, true> : k_q4_decode<NB, HPB, false>, dim3(d.splits, p.G * p.headBlocks, p.B), dim3(kDecWarps * 32), S::kSmem, s,
                          dim3(d.splits, 1, 1), p);
}
template <int NB>
void decode_heads(const DecodeParams& p, const DecodePlan& d, cudaStream_t s) {
    if (d.perBlock == 1) decode<NB, 1>(p, d, s); else if (d.perBlock == 2) decode<NB, 2>(p, d, s); else decode<NB, 4>(p, d, s);
}

}  // namespace

size_t q4_decode_ws_floats(const Q4AttnArgs& a) { const DecodePlan d = decode_plan(a); return d.records + d.ml + d.scores + d.owners; }

void launch_q4_decode(const Q4AttnArgs& a, cudaStream_t s) {
    const DecodePlan d = decode_plan(a);
    const float scale = (float)(1.0 / std::sqrt((double)a.hd) * 1.4426950408889634);
    float* const ml = a.ws + d.records;
    float* const scores = ml + d.ml;
    DecodeParams p = {a.qkv, a.q_off, a.k_off, a.v_off, a.ld, a.cache, a.maxSeq, d.pages, a.len, a.pos, a.cosT, a.sinT, a.maxPos, a.out, a.ldo, a.H, a.G,
                      a.H / a.G, d.headBlocks, scale, a.acc, a.accOut, d.scores ? scores : nullptr, a.ws, ml, reinterpret_cast<int*>(scores + d.scores), a.B,
                      a.early, g_dev_error};
    if (a.hd == 128) decode_heads<4>(p, d, s); else if (a.hd == 64) decode_heads<2>(p, d, s); else decode_heads<1>(p, d, s);
    if (!d.stream) return;
    FinishParams f = {a.len, a.pos, a.maxSeq, a.maxPos, d.pages, p.records, p.ml, p.owners, p.scores, a.acc, a.accOut, a.out, a.ldo,
                      a.H, a.G, a.H / a.G, d.headBlocks, d.perBlock, a.hd};
    launch_k(k_q4_finish, dim3(f.ratio + (p.scores != nullptr ? (a.maxSeq + kFinishRows - 1) / kFinishRows : 0), a.G, a.B), dim3(256), 0, s, true, f);
}

}  // namespace dj
