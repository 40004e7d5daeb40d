// Rows into the 4-bit cache and out of it: the append of projected keys and values, row store and load, and the eviction of rows by their
// accumulated attention weight.  The format stands in q4_cache.cuh.
#include <algorithm>

#include "kernels.h"
#include "q4_cache.cuh"

namespace dj {
namespace {

// ───────────── rows in ─────────────
// Row m of the source is token t of sequence b: m = b·T + t, or (starts) the packed row that lies in starts[b] … starts[b + 1].  A row of a head is
// 8·NB lanes of four values.  Bound by the bytes: 8·hd read and 1.125·hd written per row and head.
struct AppendParams {
    const float* src; int k_off, v_off, ld;
    unsigned char* cache; int maxSeq, pages;
    const float* starts; const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    int B, G, T, M;
};

// The sequence that packed row m belongs to (the first, should ranges overlap), or -1; whole warps call it.
__device__ __forceinline__ int sequence_of(const float* starts, int B, int M, int m, int lane, int& first, int& tokens) {
    for (int b0 = 0; b0 < B; b0 += 32) {
        const int b = b0 + lane;
        int from = 0, to = 0;
        if (b < B) { from = max(0, (int)starts[b]); to = min(M, (int)starts[b + 1]); }
        const unsigned hit = __ballot_sync(0xffffffffu, b < B && m >= from && m < to);
        if (hit) {
            const int l = __ffs(hit) - 1;
            first = __shfl_sync(0xffffffffu, from, l);
            tokens = __shfl_sync(0xffffffffu, to, l) - first;
            return b0 + l;
        }
    }
    return -1;
}

template <int NB>
__global__ void __launch_bounds__(256) k_q4_append(const AppendParams p) {
    constexpr int LPR = 8 * NB, RPW = 32 / LPR;          // lanes of a row, rows of a warp
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = blockIdx.x;
    int first = 0, tokens = p.T, b;
    if (p.starts != nullptr) {
        b = sequence_of(p.starts, p.B, p.M, m, lane, first, tokens);
        if (b < 0) return;
    } else {
        b = m / p.T;
        first = b * p.T;
    }
    const int t = m - first, len = (int)p.len[b], pos = p.pos != nullptr ? (int)p.pos[b] : 0;
    if (t >= q4_room(tokens, len, p.maxSeq, pos, p.pos != nullptr ? p.maxPos : 0x7fffffff)) return;
    const int row = len + t, e = lane % LPR;
    const float* src = p.src + (size_t)m * p.ld;
    float2 c = make_float2(1.0f, 1.0f), s = make_float2(0.0f, 0.0f);
    if (p.cosT != nullptr) {
        const size_t at = (size_t)(pos + t) * (16 * NB) + 2 * e;
        c = *reinterpret_cast<const float2*>(p.cosT + at); s = *reinterpret_cast<const float2*>(p.sinT + at);
    }
    for (int i = warp * RPW + lane / LPR; i - lane / LPR < 2 * p.G; i += 8 * RPW) {      // keys of all heads, then their values
        const bool on = i < 2 * p.G, value = i >= p.G;
        const int g = value ? i - p.G : i;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (on) x = *reinterpret_cast<const float4*>(src + (value ? p.v_off : p.k_off) + g * (32 * NB) + 4 * e);
        if (!value && p.cosT != nullptr) x = q4_rotate(x, c, s);
        unsigned char* page = p.cache + (((size_t)b * p.G + g) * p.pages + row / kQ4Page) * Q4Page<NB>::kBytes;
        q4_put_row<NB>(page, row % kQ4Page, value, e, x, on);
    }
}

// ───────────── rows out ─────────────
// Values of rows at[b] … of every head → [B][G][T][hd], as far as end[b]; other rows of the outputs stay as they are.
struct LoadParams {
    const unsigned char* cache; int maxSeq, pages;
    const float* at; const float* end; float* k; float* v; int B, G, T;
};
template <int NB>
__global__ void __launch_bounds__(256) k_q4_load(const LoadParams p) {
    constexpr int LPR = 8 * NB;                          // lanes of a row, four values each
    pdl_wait();
    pdl_launch_dependents();
    const int e = threadIdx.x % LPR, bg = blockIdx.y, b = bg / p.G;
    const int at = p.at != nullptr ? (int)p.at[b] : 0, end = min(p.maxSeq, p.end != nullptr ? (int)p.end[b] : p.maxSeq);
    if (at < 0) return;
    const int j = e >> 3, t = e & 3, shift = (e & 4);    // the four values are one nibble of each byte of word (t, j)
    for (int i = blockIdx.x * (256 / LPR) + threadIdx.x / LPR; i < p.T && i < end - at; i += gridDim.x * (256 / LPR)) {
        const int row = at + i, r = row % kQ4Page;
        const unsigned char* page = p.cache + ((size_t)bg * p.pages + row / kQ4Page) * Q4Page<NB>::kBytes;
        const size_t to = ((size_t)bg * p.T + i) * (32 * NB) + 4 * e;
#pragma unroll
        for (int value = 0; value < 2; value++) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(page + (value ? Q4Page<NB>::kV : 0) + Q4Page<NB>::word(r, t, j));
            const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(page + (value ? Q4Page<NB>::kVs : Q4Page<NB>::kKs) + (r * NB + j) * 2));
            auto val = [&](int k) { return (float)q4_code(w, 8 * k + shift) * s; };
            *reinterpret_cast<float4*>((value ? p.v : p.k) + to) = make_float4(val(0), val(1), val(2), val(3));
        }
    }
}

// ───────────── eviction ─────────────
// One block per sequence and head.  The weight of the last row that stays is found by radix selection (four passes of eight bits over an
// order-preserving map of the floats, NaN below all), then the rows move in order: the i-th kept row is never before row i, so a block that reads
// a run of rows before it writes it may work in place.
struct EvictParams {
    const unsigned char* src; int srcMax, srcPages;
    unsigned char* dst; int dstMax, dstPages;
    const float* len; const float* acc; float* accOut; float* lenOut; float* kept;
    int G, budget, recent;
};

// larger weights → larger numbers; -0 counts as 0, NaN as the least
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 256;
template <int NB>
__global__ void __launch_bounds__(kEvictThreads) k_q4_evict(const EvictParams p) {
    constexpr int kRowWords = 4 * NB;                    // code words of a row
    __shared__ unsigned s_hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_scan[kEvictThreads / 32], s_from[kEvictThreads];
    __shared__ float s_weight[kEvictThreads];
    pdl_wait();
    pdl_launch_dependents();
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t bg = (size_t)b * p.G + g;
    const int n = min(max((int)p.len[b], 0), p.srcMax), stay = min(n, p.budget), recent = min(p.recent, stay), top = stay - recent, old = n - recent;
    const float* const acc = p.acc + bg * p.srcMax;
    // the key of the last old row that stays, and how many of the rows with that key do
    uint32_t prefix = 0;
    int need = top;
    if (top > 0 && top < old) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            s_hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < old; i += kEvictThreads) {
                const uint32_t key = weight_key(acc[i]);
                if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s_hist[key >> shift & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                while (d > 0 && (int)s_hist[d] < need) need -= s_hist[d--];
                s_prefix = prefix | (uint32_t)d << shift;
                s_need = need;
            }
            __syncthreads();
            prefix = s_prefix; need = s_need;
            __syncthreads();
        }
    }
    const bool all = top == old;
    // in order, a run of rows at a time: which stay, and where they go
    int at = 0, ties = 0;                                // rows placed, rows of the threshold's key met
    for (int i0 = 0; i0 < n; i0 += kEvictThreads) {
        const int i = i0 + tid;
        float w = 0.0f;
        bool over = false, tie = false;
        if (i < n) {
            w = acc[i];
            const uint32_t key = weight_key(w);
            over = i >= old || all || (top > 0 && key > prefix);
            tie = !over && top > 0 && key == prefix;
        }
        auto rank = [&](bool flag, int& total) {         // flags of the threads before this one, and of all
            const unsigned m = __ballot_sync(0xffffffffu, flag);
            if (lane == 0) s_scan[warp] = __popc(m);
            __syncthreads();
            int before = __popc(m & ((1u << lane) - 1)), sum = 0;
#pragma unroll
            for (int k = 0; k < kEvictThreads / 32; k++) { if (k < warp) before += s_scan[k]; sum += s_scan[k]; }
            __syncthreads();
            total = sum;
            return before;
        };
        int met, found;
        const int tieRank = ties + rank(tie, met);
        ties += met;
        const bool keep = over || (tie && tieRank < need);
        const int place = rank(keep, found);
        if (keep) { s_from[place] = i; s_weight[place] = w; }
        __syncthreads();
        // the run's rows: all reads come before the writes
        for (int base = 0; base < found; base += kEvictThreads / 8) {
            const int r = base + tid / 8, c = tid % 8;   // eight threads a row: half of a K or V row's words and scales each
            constexpr int kPart = kRowWords / 4 > 0 ? kRowWords / 4 : 1;
            uint32_t words[kPart];
            unsigned short scale = 0;
            const bool value = c >= 4;
            const int t = c & 3;
            const bool on = r < found;
            if (on) {
                const int from = s_from[r];
                const unsigned char* page = p.src + (bg * p.srcPages + from / kQ4Page) * Q4Page<NB>::kBytes;
                const unsigned char* piece = page + (value ? Q4Page<NB>::kV : 0) + Q4Page<NB>::word(from % kQ4Page, t, 0);
#pragma unroll
                for (int j = 0; j < NB; j++) words[j] = *reinterpret_cast<const uint32_t*>(piece + 4 * j);
                if (t < NB) scale = *reinterpret_cast<const unsigned short*>(page + (value ? Q4Page<NB>::kVs : Q4Page<NB>::kKs) + (from % kQ4Page * NB + t) * 2);
            }
            __syncthreads();
            if (on) {
                const int to = at + r;
                unsigned char* page = p.dst + (bg * p.dstPages + to / kQ4Page) * Q4Page<NB>::kBytes;
                unsigned char* piece = page + (value ? Q4Page<NB>::kV : 0) + Q4Page<NB>::word(to % kQ4Page, t, 0);
#pragma unroll
                for (int j = 0; j < NB; j++) *reinterpret_cast<uint32_t*>(piece + 4 * j) = words[j];
                if (t < NB) *reinterpret_cast<unsigned short*>(page + (value ? Q4Page<NB>::kVs : Q4Page<NB>::kKs) + (to % kQ4Page * NB + t) * 2) = scale;
                if (c == 0) {
                    p.accOut[bg * p.dstMax + to] = s_weight[r];
                    if (p.kept != nullptr) p.kept[bg * p.budget + to] = (float)s_from[r];
                }
            }
        }
        __syncthreads();
        at += found;
    }
    if (g == 0 && tid == 0) p.lenOut[b] = (float)stay;
}

template <int NB> void append(const AppendParams& p, cudaStream_t s) { launch_k(k_q4_append<NB>, dim3(p.M), dim3(256), 0, s, true, p); }
template <int NB> void load(const LoadParams& p, cudaStream_t s) {
    const int per = 256 / (8 * NB), blocks = std::min((p.T + per - 1) / per, std::max(1, 16 * g_num_sms / (p.B * p.G)));
    launch_k(k_q4_load<NB>, dim3(blocks, p.B * p.G), dim3(256), 0, s, true, p);
}
template <int NB> void evict(const EvictParams& p, int B, cudaStream_t s) { launch_k(k_q4_evict<NB>, dim3(p.G, B), dim3(kEvictThreads), 0, s, true, p); }

}  // namespace

size_t q4_plane_bytes(int B, int G, int maxSeq, int hd) { return (size_t)B * G * ((maxSeq + kQ4Page - 1) / kQ4Page) * kQ4PageBytes * (hd / 32); }

void launch_q4_append(const Q4AttnArgs& a, int T, cudaStream_t s) {
    AppendParams p = {a.qkv, a.k_off, a.v_off, a.ld, a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.starts, a.len, a.pos, a.cosT, a.sinT, a.maxPos, a.B, a.G, T, a.M};
    if (a.hd == 128) append<4>(p, s); else if (a.hd == 64) append<2>(p, s); else append<1>(p, s);
}
void launch_q4_load(const Q4LoadArgs& a, cudaStream_t s) {
    if (a.T == 0) return;
    LoadParams p = {a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.at, a.end, a.k, a.v, a.B, a.G, a.T};
    if (a.hd == 128) load<4>(p, s); else if (a.hd == 64) load<2>(p, s); else load<1>(p, s);
}
void launch_q4_evict(const Q4EvictArgs& a, cudaStream_t s) {
    EvictParams p = {a.src, a.srcMax, (a.srcMax + kQ4Page - 1) / kQ4Page, a.dst, a.dstMax, (a.dstMax + kQ4Page - 1) / kQ4Page,
                     a.len, a.acc, a.accOut, a.lenOut, a.kept, a.G, a.budget, a.recent};
    if (a.hd == 128) evict<4>(p, a.B, s); else if (a.hd == 64) evict<2>(p, a.B, s); else evict<1>(p, a.B, s);
}

}  // namespace dj
