// Causal attention over the 4-bit cache: one token per sequence, or packed prompts of different lengths.
//
// A warp per query row and head walks the cached rows with the running maximum and sum of the softmax in fp32; a lane holds NB dims of its
// head in each 32-dim block.  The weights of rows that are asked for are added up by a second kernel from the rows' maxima and sums.
#include <cmath>

#include "kernels.h"
#include "q4_cache.cuh"

namespace dj {
namespace {

struct RowsParams {
    const float* qkv; int q_off, ld;
    const unsigned char* cache; int maxSeq, pages;
    const float* starts; const float* len; const float* pos; const float* cosT; const float* sinT; int maxPos;
    float* out; int ldo; int B, H, G, M; float scale;
    float* stats;                               // [M][H] maximum and sum of every row's softmax, or null
    const float* acc; float* accOut; int window;
};

// Sequence b's first packed row and number of tokens.
__device__ __forceinline__ void rows_of(const RowsParams& p, int b, int& first, int& tokens) {
    if (p.starts == nullptr) { first = b; tokens = 1; return; }
    first = max(0, (int)p.starts[b]);
    tokens = max(0, min(p.M, (int)p.starts[b + 1]) - first);
}

template <int NB>
__device__ __forceinline__ float dim_of(const unsigned char* page, int r, int j, int lane, bool value) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(page + (value ? Q4Page<NB>::kV : 0) + Q4Page<NB>::word(r, lane >> 2 & 3, j));
    const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(page + (value ? Q4Page<NB>::kVs : Q4Page<NB>::kKs) + (r * NB + j) * 2));
    return (float)q4_code(w, 8 * (lane & 3) + (lane >> 4) * 4) * s;          // dim 32j + lane
}

template <int NB>
__device__ __forceinline__ void query(const RowsParams& p, int m, int h, int position, int lane, float (&q)[NB]) {
    const float* row = p.qkv + (size_t)m * p.ld + p.q_off + h * (32 * NB);
#pragma unroll
    for (int j = 0; j < NB; j++) {
        const int d = 32 * j + lane;
        const float x = row[d], other = row[d ^ 1], c = p.cosT[(size_t)position * (16 * NB) + d / 2], s = p.sinT[(size_t)position * (16 * NB) + d / 2];
        q[j] = (d & 1 ? other * s + x * c : x * c - other * s) * p.scale;
    }
}

template <int NB>
__global__ void __launch_bounds__(128) k_q4_rows(const RowsParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, h = blockIdx.y, m = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (m >= p.M) return;
    int b = 0, first = 0, tokens = 0;
    for (; b < p.B; b++) {
        rows_of(p, b, first, tokens);
        if (m >= first && m < first + tokens) break;
    }
    if (b == p.B) return;
    const int t = m - first, len = (int)p.len[b], pos = (int)p.pos[b];
    if (t >= q4_room(tokens, len, p.maxSeq, pos, p.maxPos)) return;
    float q[NB], o[NB] = {}, top = -INFINITY, sum = 0.0f;
    query<NB>(p, m, h, pos + t, lane, q);
    const int g = h / (p.H / p.G);
    for (int i = 0; i <= len + t; i++) {
        const unsigned char* page = p.cache + (((size_t)b * p.G + g) * p.pages + i / kQ4Page) * Q4Page<NB>::kBytes;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; j++) dot = fmaf(q[j], dim_of<NB>(page, i % kQ4Page, j, lane, false), dot);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, k);
        const float now = fmaxf(top, dot), f = expf(top - now), w = expf(dot - now);
        sum = sum * f + w;
#pragma unroll
        for (int j = 0; j < NB; j++) o[j] = fmaf(w, dim_of<NB>(page, i % kQ4Page, j, lane, true), o[j] * f);
        top = now;
    }
#pragma unroll
    for (int j = 0; j < NB; j++) p.out[(size_t)m * p.ldo + h * (32 * NB) + 32 * j + lane] = o[j] / sum;
    if (p.stats != nullptr && lane == 0) { p.stats[((size_t)m * p.H + h) * 2] = top; p.stats[((size_t)m * p.H + h) * 2 + 1] = sum; }
}

// acc of one cached row and head: what it was, and the softmax weights that the window's queries give it
template <int NB>
__global__ void __launch_bounds__(128) k_q4_weights(const RowsParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, g = blockIdx.y, b = blockIdx.z, i = blockIdx.x * 4 + (threadIdx.x >> 5);
    int first, tokens;
    rows_of(p, b, first, tokens);
    const int len = (int)p.len[b], pos = (int)p.pos[b], room = q4_room(tokens, len, p.maxSeq, pos, p.maxPos), R = p.H / p.G;
    if (len < 0 || len >= p.maxSeq || pos < 0 || pos >= p.maxPos || i >= len + room) return;
    const unsigned char* page = p.cache + (((size_t)b * p.G + g) * p.pages + i / kQ4Page) * Q4Page<NB>::kBytes;
    const size_t at = ((size_t)b * p.G + g) * p.maxSeq + i;
    float add = 0.0f;
    for (int t = max(0, room - p.window); t < room; t++) {
        if (i > len + t) continue;
        for (int r = 0; r < R; r++) {
            const int h = g * R + r;
            float q[NB], dot = 0.0f;
            query<NB>(p, first + t, h, pos + t, lane, q);
#pragma unroll
            for (int j = 0; j < NB; j++) dot = fmaf(q[j], dim_of<NB>(page, i % kQ4Page, j, lane, false), dot);
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, k);
            const float* st = p.stats + ((size_t)(first + t) * p.H + h) * 2;
            add += expf(dot - st[0]) / st[1];
        }
    }
    if (lane == 0) p.accOut[at] = (i < len ? p.acc[at] : 0.0f) + add;
}

template <int NB>
void rows(const RowsParams& p, cudaStream_t s) {
    launch_k(k_q4_rows<NB>, dim3((p.M + 3) / 4, p.H), dim3(128), 0, s, true, p);
    if (p.accOut != nullptr) launch_k(k_q4_weights<NB>, dim3((p.maxSeq + 3) / 4, p.G, p.B), dim3(128), 0, s, true, p);
}

}  // namespace

size_t q4_attn_ws_floats(const Q4AttnArgs& a) { return a.accOut != nullptr ? (size_t)a.M * a.H * 2 : 0; }

void launch_q4_attn(const Q4AttnArgs& a, cudaStream_t s) {
    if (a.M == 0) return;
    launch_q4_append(a, 1, s);
    RowsParams p = {a.qkv, a.q_off, a.ld, a.cache, a.maxSeq, (a.maxSeq + kQ4Page - 1) / kQ4Page, a.starts, a.len, a.pos, a.cosT, a.sinT, a.maxPos,
                    a.out, a.ldo, a.B, a.H, a.G, a.M, (float)(1.0 / std::sqrt((double)a.hd)), a.accOut != nullptr ? a.ws : nullptr, a.acc, a.accOut, a.window};
    if (a.hd == 128) rows<4>(p, s); else if (a.hd == 64) rows<2>(p, s); else rows<1>(p, s);
}

}  // namespace dj
