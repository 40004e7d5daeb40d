// Rows into the 4-bit cache and out of it: the append of projected keys and values, row store and load, and the eviction of rows by their
// accumulated attention weight.  The format stands in q4_cache.cuh.
#include <algorithm>

#include "kernels.h"
#include "q4_cache.cuh"

namespace dj {
namespace {

// ───────────── rows in ─────────────
// Row m of the source is token t of sequence b: m = b·T + t, or (starts) the packed row that lies in starts[b] … starts[b + 1].  A row of a head is
// 4·NB lanes of eight values, a word of the page each.  The bytes are 8·hd read and 1.125·hd written per row and head.  2048 rows of 32 heads of 128: 20 µs where
// the bytes take 12 (with four values to a lane 27); no unit is at its limit (64 % of the issue slots, ALU 48 %): the loads' latency and the instructions for the codes.
struct AppendParams {
    const float* src; int k_off, v_off, ld;
    unsigned char* cache; int maxSeq, pages;
    const float* starts; const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    int B, G, T, M, share;                               // share: warps of a row (a power of two)
};

// The sequence that packed row m belongs to (the first, should ranges overlap), or -1; whole warps call it.
__device__ __forceinline__ int sequence_of(const float* starts, int B, int M, int m, int lane, int& first, int& tokens) {
    for (int b0 = 0; b0 < B; b0 += 32) {
        const int b = b0 + lane;
        int from = 0, n = 0;
        if (b < B) n = q4_rows(starts[b], starts[b + 1], M, from);
        const unsigned hit = __ballot_sync(0xffffffffu, m >= from && m - from < n);
        if (hit) {
            const int l = __ffs(hit) - 1;
            first = __shfl_sync(0xffffffffu, from, l);
            tokens = __shfl_sync(0xffffffffu, n, l);
            return b0 + l;
        }
    }
    return -1;
}

template <int NB>
__global__ void __launch_bounds__(256) k_q4_append(const AppendParams p) {
    constexpr int LPR = 4 * NB, RPW = 32 / LPR;          // lanes of a row, rows of a warp
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, at = blockIdx.x * 8 + (threadIdx.x >> 5), m = at / p.share, part = at - m * p.share;
    if (m >= p.M) return;
    int first = 0, tokens = p.T, b;
    if (p.starts != nullptr) {
        b = sequence_of(p.starts, p.B, p.M, m, lane, first, tokens);
        if (b < 0) return;
    } else {
        b = m / p.T;
        first = b * p.T;
    }
    const int t = m - first, len = q4_int(p.len[b]), pos = p.pos != nullptr ? q4_int(p.pos[b]) : 0;
    if (t >= q4_room(tokens, len, p.maxSeq, pos, p.pos != nullptr ? p.maxPos : 0x7fffffff)) return;
    const int row = len + t, f = lane % LPR, at0 = (f >> 2) * 32 + (f & 3) * 4;      // this lane's values: at0 … at0 + 3, and 16 on
    const float* src = p.src + (size_t)m * p.ld;
    float2 c[2] = {{1.0f, 1.0f}, {1.0f, 1.0f}}, s[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    if (p.cosT != nullptr)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const size_t at = (size_t)(pos + t) * (16 * NB) + (at0 >> 1) + 8 * h;
            c[h] = *reinterpret_cast<const float2*>(p.cosT + at); s[h] = *reinterpret_cast<const float2*>(p.sinT + at);
        }
    // keys of all heads, then their values, four rows of a warp at a time: their loads go out together
    constexpr int kAhead = 4;
    const size_t plane = (size_t)p.pages * Q4Page<NB>::kBytes;
    unsigned char* const pages = p.cache + (size_t)b * p.G * plane + (size_t)(row / kQ4Page) * Q4Page<NB>::kBytes;
    const int in = row % kQ4Page;
#pragma unroll 1
    for (int i0 = part * RPW; i0 < 2 * p.G; i0 += p.share * RPW * kAhead) {
        float4 x[kAhead][2];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int i = i0 + k * p.share * RPW + lane / LPR;
            x[k][0] = x[k][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i < 2 * p.G) {
                const float* const from = src + (i < p.G ? p.k_off + i * (32 * NB) : p.v_off + (i - p.G) * (32 * NB)) + at0;
                x[k][0] = *reinterpret_cast<const float4*>(from); x[k][1] = *reinterpret_cast<const float4*>(from + 16);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            if (i0 + k * p.share * RPW >= 2 * p.G) break;
            const int i = i0 + k * p.share * RPW + lane / LPR, g = i < p.G ? i : i - p.G;
            if (i < p.G && p.cosT != nullptr)
#pragma unroll
                for (int h = 0; h < 2; h++) x[k][h] = q4_rotate(x[k][h], c[h], s[h]);
            q4_put_words<NB>(pages + g * plane, in, i >= p.G, f, x[k][0], x[k][1], i < 2 * p.G);
        }
    }
}

// ───────────── rows out ─────────────
// Values of rows at[b] … of every head → [B][G][T][hd], as far as end[b]; other rows of the outputs stay as they are.
struct LoadParams {
    const unsigned char* cache; int maxSeq, pages;
    const float* at; const float* end; float* k; float* v; int B, G, T, share;      // share: blocks of a head
};
// A lane takes a word: four values and the four 16 on.  Bound by the writes (16 × 32 heads × 1024 rows of 128: 100 µs for 613 MB in and out; 104 with a
// lane to four values).
template <int NB>
__global__ void __launch_bounds__(256) k_q4_load(const LoadParams p) {
    constexpr int LPR = 4 * NB, AHEAD = 4;               // lanes of a row; rows whose loads go out together
    pdl_wait();
    pdl_launch_dependents();
    const int e = threadIdx.x % LPR, bg = blockIdx.x / p.share, b = bg / p.G;
    const int at = p.at != nullptr ? q4_int(p.at[b]) : 0, end = min(p.maxSeq, p.end != nullptr ? q4_int(p.end[b]) : p.maxSeq);
    if (at < 0) return;
    const int j = e >> 2, t = e & 3;
    const unsigned char* const plane = p.cache + (size_t)bg * p.pages * Q4Page<NB>::kBytes;
    const size_t out = (size_t)bg * p.T * (32 * NB) + 32 * j + 4 * t;
    const int rows = min(p.T, end - at), step = p.share * (256 / LPR);
#pragma unroll 1
    for (int i0 = ((int)blockIdx.x - bg * p.share) * (256 / LPR) + threadIdx.x / LPR; i0 < rows; i0 += AHEAD * step) {
        uint32_t w[AHEAD][2];
        unsigned short scale[AHEAD][2];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int row = at + min(i0 + k * step, rows - 1), r = row % kQ4Page;
            const unsigned char* page = plane + (size_t)(row / kQ4Page) * Q4Page<NB>::kBytes;
#pragma unroll
            for (int value = 0; value < 2; value++) {
                w[k][value] = *reinterpret_cast<const uint32_t*>(page + (value ? Q4Page<NB>::kV : 0) + Q4Page<NB>::word(r, t, j));
                scale[k][value] = *reinterpret_cast<const unsigned short*>(page + (value ? Q4Page<NB>::kVs : Q4Page<NB>::kKs) + (r * NB + j) * 2);
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (i0 + k * step < rows) {
                const size_t to = out + (size_t)(i0 + k * step) * (32 * NB);
#pragma unroll
                for (int value = 0; value < 2; value++) {
                    const float s = __uint_as_float((uint32_t)scale[k][value] << 16);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        auto val = [&](int n) { return (float)q4_code(w[k][value], 8 * n + 4 * h) * s; };
                        __stcs(reinterpret_cast<float4*>((value ? p.v : p.k) + to + 16 * h), make_float4(val(0), val(1), val(2), val(3)));
                    }
                }
            }
    }
}

// ───────────── eviction ─────────────
// A block per sequence and head finds the weight of the last row that stays by radix selection (11, 11 and 10 bits of an order-preserving map of the
// floats, NaN below all), and lists the rows that stay, in order; their weights move on the way.  Another kernel moves the rows: eight rows of a warp
// at a time, so that what it writes is contiguous.  In place the rows go through the workspace: blocks that move rows of one head run in any order.
// Bound by latency for few heads (32 heads, 2048 rows to 1024: 8 and 4 µs), for many by the integer pipe (512 heads, 4096 rows: 29 µs) and the rows' bytes (27 µs).
struct EvictParams {
    const float* len; int srcMax, dstMax;
    const float* acc; float* accOut; float* lenOut; float* kept; int* list;
    int G, budget, recent;
};

// larger weights → larger numbers; -0 counts as 0, NaN as the least
__device__ __forceinline__ uint32_t weight_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    return w != w ? 0u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

constexpr int kEvictThreads = 512, kEvictBins = 2048;
__global__ void __launch_bounds__(kEvictThreads) k_q4_select(const EvictParams p) {
    __shared__ int s_bins[kEvictBins];
    __shared__ int s_scan[kEvictThreads / 32], s_prefix, s_need;
    pdl_wait();
    pdl_launch_dependents();
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t bg = (size_t)b * p.G + g;
    const int n = min(max(q4_int(p.len[b]), 0), p.srcMax), stay = min(n, p.budget), recent = min(p.recent, stay), top = stay - recent, old = n - recent;
    const float* const acc = p.acc + bg * p.srcMax;
    int* const list = p.list + bg * p.budget;
    auto before = [&](int mine, int& total) {            // sum over the threads before this one, and over all
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
        if (lane == 31) s_scan[warp] = upto;
        __syncthreads();
        int sum = upto - mine;
        total = 0;
#pragma unroll
        for (int k = 0; k < kEvictThreads / 32; k++) { if (k < warp) sum += s_scan[k]; total += s_scan[k]; }
        __syncthreads();
        return sum;
    };
    // the key of the last old row that stays, and how many of the rows with that key do
    uint32_t prefix = 0;
    int need = top;
    if (top > 0 && top < old) {
#pragma unroll 1
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t above = pass == 0 ? 0u : pass == 1 ? ~0u << 21 : ~0u << 10, mask = pass == 2 ? 1023u : 2047u;
            for (int i = tid; i < kEvictBins; i += kEvictThreads) s_bins[i] = 0;
            __syncthreads();
            for (int i0 = tid; i0 < old; i0 += 4 * kEvictThreads) {
                float w[4];
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] = i0 + k * kEvictThreads < old ? acc[i0 + k * kEvictThreads] : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t key = weight_key(w[k]);
                    if (i0 + k * kEvictThreads < old && (key & above) == prefix) atomicAdd(&s_bins[key >> shift & mask], 1);
                }
            }
            __syncthreads();
            // bins in falling order, four to a thread: the one in which the count reaches `need`
            int c[4], mine = 0, all;
#pragma unroll
            for (int k = 0; k < 4; k++) { c[k] = s_bins[kEvictBins - 1 - 4 * tid - k]; mine += c[k]; }
            int upto = before(mine, all);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (upto < need && upto + c[k] >= need) { s_prefix = (int)(prefix | (uint32_t)(kEvictBins - 1 - 4 * tid - k) << shift); s_need = need - upto; }
                upto += c[k];
            }
            __syncthreads();
            prefix = (uint32_t)s_prefix; need = s_need;
            __syncthreads();
        }
    }
    // in order, a run of rows at a time: which stay, and where they go
    const bool every = top == old;
    int at = 0, ties = 0;                                // rows placed, rows of the threshold's key met
#pragma unroll 1
    for (int i0 = 4 * tid; i0 - 4 * tid < n; i0 += 4 * kEvictThreads) {  // four rows to a thread
        float w[4];
        int mine = 0;                                    // rows that stay in the low half, ties in the high half (runs have 2048)
        unsigned over = 0, tie = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = i0 + k < n ? acc[i0 + k] : 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k;
            const uint32_t key = weight_key(w[k]);
            const bool stays = i < n && (i >= old || every || (top > 0 && key > prefix)), ties_ = i < n && !stays && top > 0 && key == prefix;
            over |= (unsigned)stays << k; tie |= (unsigned)ties_ << k;
            mine += (stays ? 1 : 0) + (ties_ ? 1 << 16 : 0);
        }
        int both;
        const int sums = before(mine, both), room = max(need - ties, 0);                        // room: ties of this run that stay
        int overs = sums & 0xffff, met = sums >> 16;     // of this run before this row
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool stays = over >> k & 1, ties_ = tie >> k & 1;
            if (stays || (ties_ && met < room)) {
                const int place = at + overs + min(room, met);
                list[place] = i0 + k;
                p.accOut[bg * p.dstMax + place] = w[k];  // never behind this row: the rows of this run have been read
                if (p.kept != nullptr) p.kept[bg * p.budget + place] = (float)(i0 + k);
            }
            overs += stays; met += ties_;
        }
        at += (both & 0xffff) + min(room, both >> 16);
        ties += both >> 16;
    }
    if (g == 0 && tid == 0) p.lenOut[b] = (float)stay;
}

struct MoveParams {
    const unsigned char* src; int srcPages; unsigned char* dst; int dstPages;
    const float* len; int srcMax, budget, G;
    const int* list;                                     // rows of the source in the destination's order, or null: the same
    int inPlace;                                         // rows of a sequence that keeps them all stay where they are
};
template <int NB>
__global__ void __launch_bounds__(256) k_q4_move(const MoveParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int g = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, t = lane & 3;
    const size_t bg = (size_t)b * p.G + g;
    const int n = min(max(q4_int(p.len[b]), 0), p.srcMax), stay = min(n, p.budget);
    if (p.inPlace && n <= p.budget) return;
    for (int to = (int)(blockIdx.x * 8 + (threadIdx.x >> 5)) * 8 + (lane >> 2); to < stay; to += gridDim.x * 64) {
        const int from = p.list != nullptr ? p.list[bg * p.budget + to] : to, rf = from % kQ4Page, rt = to % kQ4Page;
        const unsigned char* const s = p.src + (bg * p.srcPages + from / kQ4Page) * Q4Page<NB>::kBytes;
        unsigned char* const d = p.dst + (bg * p.dstPages + to / kQ4Page) * Q4Page<NB>::kBytes;
        uint32_t w[2][NB];
        unsigned short scale[2];
#pragma unroll
        for (int value = 0; value < 2; value++) {
            const unsigned char* const half = s + (value ? Q4Page<NB>::kV : 0);
            if constexpr (NB == 4) { const uint4 v = *reinterpret_cast<const uint4*>(half + Q4Page<NB>::word(rf, t, 0)); w[value][0] = v.x; w[value][1] = v.y; w[value][2] = v.z; w[value][3] = v.w; }
            else {
#pragma unroll
                for (int j = 0; j < NB; j++) w[value][j] = *reinterpret_cast<const uint32_t*>(half + Q4Page<NB>::word(rf, t, j));
            }
            scale[value] = t < NB ? *reinterpret_cast<const unsigned short*>(half + Q4Page<NB>::kKs + (rf * NB + t) * 2) : 0;
        }
#pragma unroll
        for (int value = 0; value < 2; value++) {
            unsigned char* const half = d + (value ? Q4Page<NB>::kV : 0);
            if constexpr (NB == 4) *reinterpret_cast<uint4*>(half + Q4Page<NB>::word(rt, t, 0)) = make_uint4(w[value][0], w[value][1], w[value][2], w[value][3]);
            else {
#pragma unroll
                for (int j = 0; j < NB; j++) *reinterpret_cast<uint32_t*>(half + Q4Page<NB>::word(rt, t, j)) = w[value][j];
            }
            if (t < NB) *reinterpret_cast<unsigned short*>(half + Q4Page<NB>::kKs + (rt * NB + t) * 2) = scale[value];
        }
    }
}

template <int NB> void append(const AppendParams& p, cudaStream_t s) { launch_k(k_q4_append<NB>, dim3((unsigned)(((long long)p.M * p.share + 7) / 8)), dim3(256), 0, s, true, p); }
template <int NB> void load(LoadParams p, cudaStream_t s) {
    const int per = 256 / (4 * NB);
    p.share = std::min((p.T + per - 1) / per, std::max(1, 16 * g_num_sms / (p.B * p.G)));
    launch_k(k_q4_load<NB>, dim3((unsigned)(p.share * p.B * p.G)), dim3(256), 0, s, true, p);
}
template <int NB> void move(const MoveParams& p, int B, cudaStream_t s) {
    const int most = std::max(1, 8 * 8 * g_num_sms / (p.G * B));         // blocks of a head: all heads' fill the chip some times over
    launch_k(k_q4_move<NB>, dim3(std::min((p.budget + 63) / 64, most), p.G, B), dim3(256), 0, s, true, p);
}
void move_rows(const MoveParams& p, int B, int hd, cudaStream_t s) {
    if (hd == 128) move<4>(p, B, s); else if (hd == 64) move<2>(p, B, s); else move<1>(p, B, s);
}

}  // namespace

size_t q4_plane_bytes(int B, int G, int maxSeq, int hd) { return (size_t)B * G * ((maxSeq + kQ4Page - 1) / kQ4Page) * kQ4PageBytes * (hd / 32); }

void launch_q4_append(const Q4AttnArgs& a, int T, cudaStream_t s) {
    AppendParams p = {a.qkv, a.k_off, a.v_off, a.ld, a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.starts, a.len, a.pos, a.cosT, a.sinT, a.maxPos, a.B, a.G, T, a.M, 1};
    // A warp takes some sixteen keys and values of a row, so that its place is looked up seldom (8848 rows of 8 heads of 128: 27 µs with one warp to a row,
    // 31 with four; 2048 of 32 heads: 29 with one, 26 with four); fewer where there are few rows (16 of 32 heads: 25.6 with one, 12 with sixteen).
    while (p.share < 16 && (p.G / p.share >= 16 || (long long)a.M * p.share < 24 * g_num_sms)) p.share *= 2;
    if (a.hd == 128) append<4>(p, s); else if (a.hd == 64) append<2>(p, s); else append<1>(p, s);
}
void launch_q4_load(const Q4LoadArgs& a, cudaStream_t s) {
    if (a.T == 0) return;
    LoadParams p = {a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.at, a.end, a.k, a.v, a.B, a.G, a.T, 1};
    if (a.hd == 128) load<4>(p, s); else if (a.hd == 64) load<2>(p, s); else load<1>(p, s);
}
// In place: the rows that stay, in pages as well.  The list of rows follows.
static size_t evict_pages_floats(const Q4EvictArgs& a) { return a.src == a.dst ? (q4_plane_bytes(a.B, a.G, a.budget, a.hd) + 3) / 4 : 0; }
size_t q4_evict_ws_floats(const Q4EvictArgs& a) { return evict_pages_floats(a) + (size_t)a.B * a.G * a.budget; }
void launch_q4_evict(const Q4EvictArgs& a, cudaStream_t s) {
    int* const list = reinterpret_cast<int*>(a.ws + evict_pages_floats(a));
    EvictParams p = {a.len, a.srcMax, a.dstMax, a.acc, a.accOut, a.lenOut, a.kept, list, a.G, a.budget, a.recent};
    launch_k(k_q4_select, dim3(a.G, a.B), dim3(kEvictThreads), 0, s, true, p);
    auto pages = [](int rows) { return (rows + kQ4Page - 1) / kQ4Page; };
    const bool inPlace = a.src == a.dst;
    unsigned char* const between = reinterpret_cast<unsigned char*>(a.ws);
    MoveParams m = {a.src, pages(a.srcMax), inPlace ? between : a.dst, pages(inPlace ? a.budget : a.dstMax), a.len, a.srcMax, a.budget, a.G, list, inPlace};
    move_rows(m, a.B, a.hd, s);
    if (!inPlace) return;
    m.src = between; m.srcPages = pages(a.budget); m.dst = a.dst; m.dstPages = pages(a.dstMax); m.list = nullptr;
    move_rows(m, a.B, a.hd, s);
}

}  // namespace dj
