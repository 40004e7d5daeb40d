// One new token per sequence over the 4-bit cache: rotation, append, attention and accumulated weights.
//
// grid (splits, heads of the cache × blocks of query heads, sequences).  A warp streams pages of 32 rows through a ring of its own, one bulk copy
// each, and keeps the running maximum and sum of the softmax in fp32.  Both products run on the integer tensor pipe, exactly:
//   scores   A = 16 rows × 32 dims of int8 codes (a masked page word is an operand register), B = the query in fixed point, 23 bits of its largest
//            value, as three signed base-256 digits.  A 32-dim block's integer sums are multiplied by the row's scale in fp32.
//   values   A = 16 dims × 32 rows (a byte transpose of four rows' words), B = weight × scale of the row and block, in fixed point of the page's
//            largest such product, three digits again.
// Columns 2t and 2t + 1 of B are digit t of two heads, so a lane sees one digit of up to two heads per tile and the digits meet in two shuffles.
// The new row is quantized by the warp that holds its page, into the page's copy in shared memory and into the cache: later steps read what this one did.
// Up to eight splits are a cluster, which exchanges maxima, sums and unnormalised rows through distributed shared memory; more leave them in the
// workspace for k_q4_finish.  Weights are added up from the scores, which wait in the workspace until the row's maximum and sum are known.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "q4_cache.cuh"
#include "tc_common.cuh"

namespace dj {
namespace {

constexpr int kDecWarps = 4;
constexpr int kDecCluster = 8;                 // up to so many splits are a cluster
constexpr int kDecMaxSplits = 128;
constexpr int kErrQ4Page = 334;                // device error code: a page never arrived
constexpr int kDecSpin = 1 << 22;

struct DecodeParams {
    const float* qkv; int q_off, k_off, v_off, ld;
    unsigned char* cache; int maxSeq, pages;
    const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    float* out; int ldo; int H, G, ratio, headBlocks; float scale;      // scale: 1/sqrt(hd) · log2(e)
    const float* acc; float* accOut;
    float* scores;                             // [B][H][pages · 32], log2 units; null: weights are not wanted
    float* partial;                            // [B][H][splits][hd + 2]: without a cluster
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
// For |x| <= most: 2^23 / 2^(exponent + 2), which brings x to fixed point below 2^22, and its inverse.  Magnitudes under 2^-100 count as nothing.
__device__ __forceinline__ float fixed_of(float most, float& back) {
    const int bits = most > 7.8886091e-31f && most < 1e36f ? (__float_as_int(most) & 0x7f800000) + 0x01000000 : 0x3f800000;
    back = __int_as_float(bits) * (1.0f / 8388608.0f);
    return most > 7.8886091e-31f ? __int_as_float(0x7f000000 - bits) * 8388608.0f : 0.0f;
}
// x · mul in fixed point → three signed base-256 digits in the low bytes
__device__ __forceinline__ uint32_t digits_of(float x, float mul) { return (uint32_t)(__float2int_rn(x * mul) + 0x808080) ^ 0x808080u; }

template <int NB> struct Words { uint32_t w[NB]; };
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
    static constexpr int HD = 32 * NB, NT = (HPB + 1) / 2;
    static constexpr int kStages = NB == 4 ? 2 : NB == 2 ? 4 : 6;
    static constexpr int kRing = kDecWarps * kStages * Q4Page<NB>::kBytes;
    static constexpr int kDigits = NB * HPB * 96;                        // of a warp: [block][head][digit][32 rows]
    static constexpr size_t kSmem = kRing + kDecWarps * kDigits + 64;    // 64: zeros for the columns without a head
};

template <int NB, int HPB, bool CLUSTER>
__global__ void __launch_bounds__(kDecWarps * 32, HPB == 4 ? 3 : 4) k_q4_decode(const DecodeParams p) {
    using S = DecodeShape<NB, HPB>;
    using Page = Q4Page<NB>;
    constexpr int HD = S::HD, NT = S::NT, kStages = S::kStages, kOut = HPB * HD;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) unsigned long long s_bar[kDecWarps * kStages];
    __shared__ __align__(16) uint32_t s_q[HPB][3][HD / 4];               // the queries' digits
    __shared__ float s_factor[HPB], s_m[kDecWarps][HPB], s_l[kDecWarps][HPB];
    __shared__ float s_ml[CLUSTER ? kDecCluster : 1][HPB][2];            // every split's maximum and sum
    __shared__ float s_red[CLUSTER ? kOut : 1];                          // this block's share of the output row, of every split
    const int split = blockIdx.x, splits = gridDim.x, g_ = blockIdx.y / p.headBlocks, hb = blockIdx.y - g_ * p.headBlocks, b = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int heads = min(HPB, p.ratio - hb * HPB), h0 = g_ * p.ratio + hb * HPB;
    if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const uint32_t bars = smem_u32(&s_bar[warp * kStages]);
    unsigned char* const ring = smem + warp * (kStages * Page::kBytes);
    unsigned char* const digits = smem + S::kRing + warp * S::kDigits;
    unsigned char* const zeros = smem + S::kRing + kDecWarps * S::kDigits;
    if (lane < kStages) mbar_init(bars + 8 * lane, 1);
    if (tid < 16) reinterpret_cast<uint32_t*>(zeros)[tid] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();

    unsigned char* const plane = p.cache + ((size_t)b * p.G + g_) * p.pages * Page::kBytes;
    int asked = 0, taken = 0, limit = kDecSpin, first = 0, end = 0;      // pages first + warp, + kDecWarps, … below end
    auto request = [&]() {
        const int pg = first + warp + asked * kDecWarps;
        if (pg < end) {
            if (lane == 0) {
                const uint32_t bar = bars + 8 * (asked % kStages);
                mbar_arrive_expect_tx(bar, Page::kBytes);
                bulk_g2s(smem_u32(ring + asked % kStages * Page::kBytes), plane + (size_t)pg * Page::kBytes, Page::kBytes, bar);
            }
            asked++;
        }
    };
    auto take = [&]() {
        const uint32_t bar = bars + 8 * (taken % kStages), parity = (taken / kStages) & 1;
        bool ready = mbar_try_wait(bar, parity);
#pragma unroll 1
        for (int spin = 0; !ready && spin < limit; spin++) ready = mbar_try_wait(bar, parity);
        if (!ready) {                             // never on a healthy device: flag it, stop waiting long, keep the control flow
            if (lane == 0) atomicCAS(p.error, 0, kErrQ4Page);
            limit = 64;
        }
        taken++;
    };
    auto slice = [&](int len) {
        const int pages = len / kQ4Page + 1, share = (pages + splits - 1) / splits;
        first = min(pages, split * share);
        end = min(pages, first + share);
    };
    int len = 0, pos = 0;
    bool there = false;
    auto place = [&]() {                          // where this sequence stands
        len = (int)__ldcg(p.len + b); pos = (int)__ldcg(p.pos + b);
        there = q4_room(1, len, p.maxSeq, pos, p.maxPos) == 1;
        if (there) slice(len);
    };
    // Behind a projection of the same stream the cached rows are complete: the first pages are asked for before the dependency wait.  A length that
    // has moved by then (never observed) drops them.
    int before = -1;
    if (p.early) {
        place();
        before = there ? len : -1;
        if (there)
#pragma unroll 1
            for (int i = 0; i < kStages; i++) request();
    }
    pdl_wait();
    pdl_launch_dependents();
    place();
    if (before >= 0 && (!there || len != before)) {
#pragma unroll 1
        while (taken < asked) take();
        __syncwarp();
        asked = taken = 0;
        before = -1;
        // the ring starts over: its barriers' phases go on from where they are
        if (lane < kStages) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bars + 8 * lane) : "memory"); mbar_init(bars + 8 * lane, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    if (!there) {                                 // the whole cluster: it shares the sequence
        if constexpr (CLUSTER) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    if (before < 0)
#pragma unroll 1
        for (int i = 0; i < kStages; i++) request();

    // queries: rotated, in fixed point of the head's largest value
    const float* const row = p.qkv + (size_t)b * p.ld;
    constexpr int LPR = 8 * NB;                   // lanes of a row of four values each
    const int e = lane % LPR;
    const size_t tab = (size_t)pos * (HD / 2) + 2 * e;
    const float2 cs = *reinterpret_cast<const float2*>(p.cosT + tab), sn = *reinterpret_cast<const float2*>(p.sinT + tab);
    for (int h = warp; h < HPB; h += kDecWarps) {
        float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (h < heads) q = q4_rotate(*reinterpret_cast<const float4*>(row + p.q_off + (h0 + h) * HD + 4 * e), cs, sn);
        float most = fmaxf(fmaxf(fabsf(q.x), fabsf(q.y)), fmaxf(fabsf(q.z), fabsf(q.w)));
        most = warp_max(most);
        float bad = (q.x + q.y + q.z + q.w) * 0.0f, back;                // NaN where the query holds an infinity or a NaN
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) bad += __shfl_xor_sync(0xffffffffu, bad, o);
        const float mul = fixed_of(most, back);
        const uint32_t u0 = digits_of(q.x, mul), u1 = digits_of(q.y, mul), u2 = digits_of(q.z, mul), u3 = digits_of(q.w, mul);
        const uint32_t t0 = __byte_perm(u0, u1, 0x5140), t1 = __byte_perm(u2, u3, 0x5140), t2 = __byte_perm(u0, u1, 0x7362), t3 = __byte_perm(u2, u3, 0x7362);
        if (lane < LPR) {
            s_q[h][2][e] = __byte_perm(t0, t1, 0x5410);
            s_q[h][1][e] = __byte_perm(t0, t1, 0x7632);
            s_q[h][0][e] = __byte_perm(t2, t3, 0x5410);
        }
        if (lane == 0) s_factor[h] = back * p.scale * (1.0f / 16.0f) + bad;
    }
    __syncthreads();
    uint32_t bq[NT][NB][2];
    float factor[HPB];                            // of this lane's digit
    const float digit = t == 0 ? 65536.0f : t == 1 ? 256.0f : t == 2 ? 1.0f : 0.0f;
    const int hc = g & 1, dc = g >> 1;            // head and digit of the B column this lane fills
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const bool on = dc < 3 && 2 * n + hc < HPB;
            bq[n][j][0] = on ? s_q[on ? 2 * n + hc : 0][on ? dc : 0][8 * j + t] : 0;
            bq[n][j][1] = on ? s_q[on ? 2 * n + hc : 0][on ? dc : 0][8 * j + 4 + t] : 0;
        }
#pragma unroll
    for (int h = 0; h < HPB; h++) factor[h] = s_factor[h] * digit;

    float m[HPB], l[HPB], acc[NT][NB][2][HPB == 1 ? 2 : 4];              // [tile of heads][block][half][row g, row g + 8 × heads]
#pragma unroll
    for (int h = 0; h < HPB; h++) { m[h] = -INFINITY; l[h] = 0.0f; }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int k = 0; k < (HPB == 1 ? 2 : 4); k++) acc[n][j][x][k] = 0.0f;
    const int key = 8 * t + g;                    // the row of a page that this lane's weights are of
    const int put = (key & 3) * 8 + (key >> 4) * 4 + ((key >> 2) & 3);   // … and their place in an operand: byte (key / 4 % 4) of word (key % 4, key / 16)
    const uint32_t pick = g & 1 ? 0x7362u : 0x5140u;
    const int rows = len + 1;

#pragma unroll 1
    for (int pg = first + warp; pg < end; pg += kDecWarps) {
        unsigned char* const page = ring + taken % kStages * Page::kBytes;
        take();
        if (pg == len / kQ4Page) {                // the new row: keys in the lower lanes first, then values
            const int r = len % kQ4Page;
#pragma unroll
            for (int value = 0; value < 2; value++) {
                float4 x = *reinterpret_cast<const float4*>(row + (value ? p.v_off : p.k_off) + g_ * HD + 4 * e);
                if (!value) x = q4_rotate(x, cs, sn);
                q4_put_row<NB>(page, r, value, e, x, lane < LPR);
                if (hb == 0) q4_put_row<NB>(plane + (size_t)pg * Page::kBytes, r, value, e, x, lane < LPR);
            }
            __syncwarp();
        }
        // scores of the page's 32 rows: rows 8k + g in s[h][k]
        float s[HPB][4];
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            uint32_t wa[NB], wb[NB];
            float sa[NB], sb[NB];
            lds_piece<NB>(wa, page + Page::word(16 * mt + g, t, 0));
            lds_piece<NB>(wb, page + Page::word(16 * mt + 8 + g, t, 0));
            lds_scales<NB>(sa, page + Page::kKs + (16 * mt + g) * NB * 2);
            lds_scales<NB>(sb, page + Page::kKs + (16 * mt + 8 + g) * NB * 2);
#pragma unroll
            for (int h = 0; h < HPB; h++) s[h][2 * mt] = s[h][2 * mt + 1] = 0.0f;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const uint32_t a[4] = {q4_low(wa[j]), q4_low(wb[j]), q4_high(wa[j]), q4_high(wb[j])};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    int d[4];
                    mma_q4(d, a, bq[n][j][0], bq[n][j][1], kMagic);
                    s[2 * n][2 * mt] = fmaf(from_magic(d[0]), sa[j], s[2 * n][2 * mt]);
                    s[2 * n][2 * mt + 1] = fmaf(from_magic(d[2]), sb[j], s[2 * n][2 * mt + 1]);
                    if constexpr (HPB > 1) {
                        s[2 * n + 1][2 * mt] = fmaf(from_magic(d[1]), sa[j], s[2 * n + 1][2 * mt]);
                        s[2 * n + 1][2 * mt + 1] = fmaf(from_magic(d[3]), sb[j], s[2 * n + 1][2 * mt + 1]);
                    }
                }
            }
        }
        const bool in = pg * kQ4Page + key < rows;
        float vs[NB], back[HPB][NB];
        lds_scales<NB>(vs, page + Page::kVs + key * NB * 2);
#pragma unroll
        for (int h = 0; h < HPB; h++) {
#pragma unroll
            for (int k = 0; k < 4; k++) {         // the digits meet: every lane of a row has its sum
                s[h][k] *= factor[h];
                s[h][k] += __shfl_xor_sync(0xffffffffu, s[h][k], 1);
                s[h][k] += __shfl_xor_sync(0xffffffffu, s[h][k], 2);
            }
            float sc = t & 2 ? (t & 1 ? s[h][3] : s[h][2]) : (t & 1 ? s[h][1] : s[h][0]);
            if (p.scores != nullptr && h < heads) p.scores[((size_t)b * p.H + h0 + h) * ((size_t)p.pages * kQ4Page) + pg * kQ4Page + key] = sc;
            sc = in ? sc : -INFINITY;
            const float now = fmaxf(m[h], warp_max(sc));
            if (now > m[h]) {                     // seldom after the first pages
                const float f = ex2(m[h] - now);
                l[h] *= f;
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        acc[h / 2][j][x][HPB == 1 ? 0 : h % 2] *= f;
                        acc[h / 2][j][x][HPB == 1 ? 1 : 2 + h % 2] *= f;
                    }
                m[h] = now;
            }
            const float w = in ? ex2(sc - m[h]) : 0.0f;
            l[h] += w;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const float x = w * vs[j];
                const float mul = fixed_of(warp_max(x), back[h][j]);
                const uint32_t u = digits_of(x, mul);
                unsigned char* const to = digits + (j * HPB + h) * 96 + put;
                to[0] = (unsigned char)(u >> 16); to[32] = (unsigned char)(u >> 8); to[64] = (unsigned char)u;
            }
        }
        __syncwarp();
        // values
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
                    if constexpr (HPB == 1) {
                        acc[0][j][x][0] = fmaf(from_magic(d[0]), back[0][j], acc[0][j][x][0]);
                        acc[0][j][x][1] = fmaf(from_magic(d[2]), back[0][j], acc[0][j][x][1]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; k++) acc[n][j][x][k] = fmaf(from_magic(d[k]), back[2 * n + (k & 1)][j], acc[n][j][x][k]);
                    }
                }
            }
        }
        __syncwarp();                             // the slot and the digits are read out
        request();
    }

    // the warp's digits meet; rows of the block's warps meet in the ring's memory, where nothing is on its way any more
    __syncthreads();
    float* const part = reinterpret_cast<float*>(smem);                  // [warp][head][HD]
#pragma unroll
    for (int h = 0; h < HPB; h++) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
        if (lane == 0) { s_m[warp][h] = m[h]; s_l[warp][h] = l[h]; }
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float a = acc[h / 2][j][x][HPB == 1 ? r : 2 * r + h % 2] * (digit * (1.0f / 16.0f));
                    a += __shfl_xor_sync(0xffffffffu, a, 1);
                    a += __shfl_xor_sync(0xffffffffu, a, 2);
                    if (t == 0) part[(warp * HPB + h) * HD + 32 * j + 16 * x + 2 * g + r] = a;
                }
    }
    __syncthreads();
    auto block_max = [&](int h) { return fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h])); };
    auto weight = [](float mine, float top) { return mine > -INFINITY ? ex2(mine - top) : 0.0f; };
    auto block_sum = [&](int h, float top) {
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) a = fmaf(s_l[w][h], weight(s_m[w][h], top), a);
        return a;
    };
    auto block_row = [&](int i, float top) {
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) a = fmaf(part[w * kOut + i], weight(s_m[w][i / HD], top), a);
        return a;
    };
    float* const orow = p.out + (size_t)b * p.ldo + h0 * HD;
    if (splits > 1 && !CLUSTER) {
        for (int i = tid; i < heads * HD; i += kDecWarps * 32)
            p.partial[(((size_t)b * p.H + h0 + i / HD) * splits + split) * (HD + 2) + i % HD] = block_row(i, block_max(i / HD));
        if (tid < heads) {
            float* const to = p.partial + (((size_t)b * p.H + h0 + tid) * splits + split) * (HD + 2) + HD;
            to[0] = block_max(tid); to[1] = block_sum(tid, block_max(tid));
        }
        return;
    }
    if (!CLUSTER) {
        for (int i = tid; i < heads * HD; i += kDecWarps * 32) { const float top = block_max(i / HD); orow[i] = block_row(i, top) / block_sum(i / HD, top); }
        if (tid < HPB) { s_ml[0][tid][0] = block_max(tid); s_ml[0][tid][1] = block_sum(tid, block_max(tid)); }
        __syncthreads();
    } else {
        __syncwarp();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // every block of the cluster is running
        const int share = kOut / splits;          // elements of the row that a block adds up
        auto put_to = [](const float* at, int rank, float x) {
            uint32_t a;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(at)), "r"(rank));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory");
        };
        for (int i = tid; i < kOut; i += kDecWarps * 32) put_to(&s_red[split * share + i % share], i / share, block_row(i, block_max(i / HD)));
        if (tid < HPB * splits) {
            const int h = tid % HPB;
            const float top = block_max(h);
            put_to(&s_ml[split][h][0], tid / HPB, top);
            put_to(&s_ml[split][h][1], tid / HPB, block_sum(h, top));
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = tid; i < share; i += kDecWarps * 32) {
            const int at = split * share + i, h = at / HD;
            float top = -INFINITY, sum = 0.0f, a = 0.0f;
            for (int r = 0; r < splits; r++) top = fmaxf(top, s_ml[r][h][0]);
            for (int r = 0; r < splits; r++) {
                const float f = weight(s_ml[r][h][0], top);
                sum = fmaf(s_ml[r][h][1], f, sum);
                a = fmaf(s_red[r * share + i], f, a);
            }
            if (h < heads) orow[at] = a / sum;
        }
    }
    if (p.scores == nullptr || p.headBlocks > 1) return;
    // this block's rows: their old weights and those of this step
    float top[HPB], inv[HPB];
#pragma unroll
    for (int h = 0; h < HPB; h++) {
        top[h] = -INFINITY;
        float sum = 0.0f;
        for (int r = 0; r < (CLUSTER ? splits : 1); r++) top[h] = fmaxf(top[h], s_ml[r][h][0]);
        for (int r = 0; r < (CLUSTER ? splits : 1); r++) sum = fmaf(s_ml[r][h][1], weight(s_ml[r][h][0], top[h]), sum);
        inv[h] = 1.0f / sum;
    }
    const size_t at = ((size_t)b * p.G + g_) * p.maxSeq, pitch = (size_t)p.pages * kQ4Page;
    for (int i = first * kQ4Page + tid; i < min(rows, end * kQ4Page); i += kDecWarps * 32) {
        float add = 0.0f;
#pragma unroll
        for (int h = 0; h < HPB; h++)
            if (h < heads) add = fmaf(ex2(p.scores[((size_t)b * p.H + h0 + h) * pitch + i] - top[h]), inv[h], add);
        p.accOut[at + i] = (i < len ? p.acc[at + i] : 0.0f) + add;
    }
}

// More splits than a cluster has, or weights of several head blocks.  Blocks (0, head of the cache, sequence) merge the splits of the group's heads,
// all blocks add up the weights of a run of rows.
struct FinishParams {
    const float* len; const float* pos; int maxSeq, maxPos, pages;
    const float* partial; int splits;
    const float* scores; const float* acc; float* accOut;
    float* out; int ldo; int H, G, ratio, hd;
};
constexpr int kFinishRows = 1024;
__global__ void __launch_bounds__(256) k_q4_finish(const FinishParams p) {
    __shared__ float s_top[64], s_inv[64];
    pdl_wait();
    pdl_launch_dependents();
    const int g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, len = (int)p.len[b], pos = (int)p.pos[b];
    if (q4_room(1, len, p.maxSeq, pos, p.maxPos) != 1) return;
    const int from = blockIdx.x * kFinishRows;
    if (blockIdx.x > 0 && from > len) return;
    const int rec = p.hd + 2;
    for (int r = warp; r < p.ratio; r += 8) {
        const float* at = p.partial + ((size_t)b * p.H + g * p.ratio + r) * p.splits * rec;
        float top = -INFINITY, sum = 0.0f;
        for (int i = lane; i < p.splits; i += 32) top = fmaxf(top, at[(size_t)i * rec + p.hd]);
        top = warp_max(top);
        for (int i = lane; i < p.splits; i += 32) { const float m = at[(size_t)i * rec + p.hd]; sum = fmaf(at[(size_t)i * rec + p.hd + 1], m > -INFINITY ? ex2(m - top) : 0.0f, sum); }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) { s_top[r] = top; s_inv[r] = 1.0f / sum; }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = tid; i < p.ratio * p.hd; i += 256) {
            const int r = i / p.hd, d = i - r * p.hd;
            const float* at = p.partial + ((size_t)b * p.H + g * p.ratio + r) * p.splits * rec;
            float a = 0.0f;
            for (int k = 0; k < p.splits; k++) {
                const float m = at[(size_t)k * rec + p.hd];
                a = fmaf(at[(size_t)k * rec + d], m > -INFINITY ? ex2(m - s_top[r]) : 0.0f, a);
            }
            p.out[(size_t)b * p.ldo + g * p.ratio * p.hd + i] = a * s_inv[r];
        }
    if (p.scores == nullptr) return;
    const size_t at = ((size_t)b * p.G + g) * p.maxSeq, pitch = (size_t)p.pages * kQ4Page;
    for (int i = from + tid; i <= min(len, from + kFinishRows - 1); i += 256) {
        float add = 0.0f;
        for (int r = 0; r < p.ratio; r++) add = fmaf(ex2(p.scores[((size_t)b * p.H + g * p.ratio + r) * pitch + i] - s_top[r]), s_inv[r], add);
        p.accOut[at + i] = (i < len ? p.acc[at + i] : 0.0f) + add;
    }
}

int heads_per_block(int ratio) { return ratio >= 3 ? 4 : ratio; }

// Splits of a sequence and head: enough blocks to fill the slots, but at least a page per warp.  Powers of two up to eight, which are clusters.
int decode_splits(int blocks, int pages) {
    const int slots = 4 * g_num_sms, most = std::max(1, (pages + kDecWarps - 1) / kDecWarps);
    int s = 1;
    while (s < kDecCluster && s * 2 <= most && blocks * s * 2 <= slots) s *= 2;
    if (s == kDecCluster && blocks * s * 2 <= slots && pages >= 64 * kDecWarps) s = std::min({kDecMaxSplits, slots / blocks, pages / (4 * kDecWarps)});
    return s;
}

template <int NB, int HPB>
void decode(const DecodeParams& p, int splits, int B, cudaStream_t s) {
    using S = DecodeShape<NB, HPB>;
    static bool attr = false;
    if (!attr) {
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_decode<NB, HPB, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        DJ_CUDA_CHECK(cudaFuncSetAttribute(k_q4_decode<NB, HPB, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        attr = true;
    }
    const bool cluster = splits > 1 && splits <= kDecCluster;
    launch_k_cluster(cluster ? k_q4_decode<NB, HPB, true> : k_q4_decode<NB, HPB, false>, dim3(splits, p.G * p.headBlocks, B), dim3(kDecWarps * 32), S::kSmem, s,
                     dim3(cluster ? splits : 1, 1, 1), p);
}
template <int NB>
void decode_heads(const DecodeParams& p, int splits, int B, cudaStream_t s) {
    const int h = heads_per_block(p.ratio);
    if (h == 1) decode<NB, 1>(p, splits, B, s); else if (h == 2) decode<NB, 2>(p, splits, B, s); else decode<NB, 4>(p, splits, B, s);
}

struct DecodePlan { int headBlocks, pages, splits; bool finish; size_t scores, partial; };
DecodePlan decode_plan(const Q4AttnArgs& a) {
    DecodePlan d;
    const int ratio = a.H / a.G;
    d.headBlocks = (ratio + heads_per_block(ratio) - 1) / heads_per_block(ratio);
    d.pages = (a.maxSeq + kQ4Page - 1) / kQ4Page;
    d.splits = decode_splits(a.B * a.G * d.headBlocks, d.pages);
    // the weights of a group's heads are added up in one place: by the kernel itself where one block has them all
    d.finish = d.splits > kDecCluster;
    if (a.accOut != nullptr && d.headBlocks > 1) { d.finish = true; d.splits = std::max(d.splits, kDecCluster + 1); }
    d.scores = a.accOut != nullptr ? (size_t)a.B * a.H * d.pages * kQ4Page : 0;
    d.partial = d.finish ? (size_t)a.B * a.H * d.splits * (a.hd + 2) : 0;
    return d;
}

}  // namespace

size_t q4_decode_ws_floats(const Q4AttnArgs& a) { const DecodePlan d = decode_plan(a); return d.scores + d.partial; }

void launch_q4_decode(const Q4AttnArgs& a, cudaStream_t s) {
    const DecodePlan d = decode_plan(a);
    const float scale = (float)(1.0 / std::sqrt((double)a.hd) * 1.4426950408889634);
    DecodeParams p = {a.qkv, a.q_off, a.k_off, a.v_off, a.ld, a.cache, a.maxSeq, d.pages, a.len, a.pos, a.cosT, a.sinT, a.maxPos, a.out, a.ldo, a.H, a.G,
                      a.H / a.G, d.headBlocks, scale, a.acc, a.accOut, d.scores ? a.ws : nullptr, a.ws + d.scores, a.early, g_dev_error};
    if (a.hd == 128) decode_heads<4>(p, d.splits, a.B, s); else if (a.hd == 64) decode_heads<2>(p, d.splits, a.B, s); else decode_heads<1>(p, d.splits, a.B, s);
    if (!d.finish) return;
    FinishParams f = {a.len, a.pos, a.maxSeq, a.maxPos, d.pages, p.partial, d.splits, p.scores, a.acc, a.accOut, a.out, a.ldo, a.H, a.G, a.H / a.G, a.hd};
    launch_k(k_q4_finish, dim3(p.scores != nullptr ? (a.maxSeq + kFinishRows - 1) / kFinishRows : 1, a.G, a.B), dim3(256), 0, s, true, f);
}

}  // namespace dj
