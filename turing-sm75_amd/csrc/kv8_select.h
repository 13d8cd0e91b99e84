// kv8_select.h -- the blocks of an 8-bit K/V cache that each query attends to, by a cheap score.
//
// With A the largest |q| of the group's heads, qc = rint(127 q / A), and a block's summary m
// (8 bits, step m_scale; see kv8_cache.h), the score is max_g sum_d qc[g][d] m[d], a whole number
// below 2^24, times m_scale: one fp32 product, so every order of summing gives the same score and
// the same choice.  A group's queries share their blocks (A does not change the order).
#pragma once
#include <climits>

#include "kv8.h"

namespace tsa {
namespace {

struct Kv8SelectArgs {
    Kv8 c;
    Rows16 q;
    const int *len, *n_new;
    float* score;      // [B][Hkv][T][nb]
    int* blocks;       // [B][Hkv][T][top]
    int T, Hq, G, top, first, recent, nb;
    int tq;            // queries of a score workgroup
};

constexpr int kKvScoreCols = 48;    // query rows (t, g) of a score workgroup at the most, or one query's heads
constexpr int kKvScoreBlocks = 128; // blocks of one

// Workgroup (queries and blocks, b Hkv + h): scores of 128 blocks, 32 a wave, for `tq` queries whose
// codes lie in LDS, by v_mfma_i32_16x16x64_i8 with the summaries as operand A straight from memory
// (lane l: block l % 16, d = 64 k + 16 (l / 16) + 0 .. 15) and 16 query rows as operand B.  Lane l
// then has 4 blocks' scores of row l % 16; the maximum over a query's heads goes through LDS.  With
// more than 48 heads a group, the rows of one query are taken 48 at a time.
template <int D>
__global__ void __launch_bounds__(256)
kv8_score_kernel(Kv8SelectArgs p) {
    typedef int int4_v __attribute__((ext_vector_type(4)));
    constexpr int kRow = D + 16, kWaveTiles = kKvScoreBlocks / 64;
    __shared__ __align__(16) signed char qs[kKvScoreCols * kRow];
    __shared__ int sc[kKvScoreCols][kKvScoreBlocks + 4];
    __shared__ int most[kKvScoreCols];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g4 = lane >> 4, n = lane & 15;
    const int parts = (p.nb + kKvScoreBlocks - 1) / kKvScoreBlocks, blk0 = (int)(blockIdx.x % parts) * kKvScoreBlocks;
    const int b = blockIdx.y / p.c.Hkv, h = blockIdx.y % p.c.Hkv, t0 = (int)(blockIdx.x / parts) * p.tq;
    // operand A first: its latency passes under the query codes'
    int page[kWaveTiles];
    int4_v m[kWaveTiles][D / 64];
    const int table_end = min(p.nb, p.c.max_blocks);
#pragma unroll
    for (int i = 0; i < kWaveTiles; ++i) {
        const int blk = blk0 + 16 * (kWaveTiles * wave + i) + n;
        page[i] = blk < table_end ? kv8_page(p.c, b, blk) : -1;
        const signed char* at = p.c.k_sum + ((size_t)max(page[i], 0) * p.c.Hkv + h) * D + 16 * g4;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) m[i][k] = *reinterpret_cast<const int4_v*>(at + 64 * k);
    }
    const Kv8Seq sq = kv8_seq(p.c, p.len, p.n_new, b, p.T);
    const int nt = min(p.tq, sq.n + sq.t0 - t0), front = sq.len - (sq.n + sq.t0);
    if (nt <= 0) return;
    if (blk0 >= min((front + t0 + nt - 1) / kKvBlock, p.nb)) return;  // no query's own block has a score
    const half_t* q = p.q.data + b * p.q.b + (long long)h * p.G * p.q.h + (long long)t0 * p.q.t;
    if (tid < nt) most[tid] = 1;
    __syncthreads();
    // max |q| of each query's group, as the bits of its fp16: infinities and NaN are at least 0x7c00.
    // Up to 48 rows stay in registers for their codes.
    constexpr int kHeld = kKvScoreCols * (D / 8) / 256 + (kKvScoreCols * (D / 8) % 256 ? 1 : 0);
    half8_t held[kHeld];
    auto load = [&](int i) {
        const int row = i / (D / 8);
        return *reinterpret_cast<const half8_t*>(q + row / p.G * p.q.t + row % p.G * p.q.h + i % (D / 8) * 8);
    };
    const int parts8 = nt * p.G * (D / 8);  // of 8 elements
#pragma unroll
    for (int j = 0; j < kHeld; ++j) held[j] = tid + 256 * j < parts8 ? load(tid + 256 * j) : half8_t{};
    auto raise = [&](int i, half8_t x) {
        const int row = i / (D / 8);
        int a = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) a = max(a, (int)(__builtin_bit_cast(unsigned short, (half_t)x[j]) & 0x7fff));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) a = max(a, __shfl_xor(a, o));  // 8 lanes are of one row
        if ((i & 7) == 0) atomicMax(&most[row / p.G], a);
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (tid + 256 * j < parts8) raise(tid + 256 * j, held[j]);
    for (int i = tid + 256 * kHeld; i < parts8; i += 256) raise(i, load(i));
    int best = INT_MIN;  // one query of many heads: the maximum over its rounds
    for (int col0 = 0; col0 < nt * p.G; col0 += kKvScoreCols) {
        const int cols = min(kKvScoreCols, nt * p.G - col0);
        __syncthreads();
        auto code = [&](int i, half8_t x) {
            const int col = i / (D / 8), row = col0 + col, big = most[row / p.G];
            // a group with an infinity or NaN has no order: all its codes are 0
            const float a = big < 0x7c00 ? (float)__builtin_bit_cast(half_t, (unsigned short)big) : 1.f, r = 1.f / a;
            unsigned y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = kv8_code(big < 0x7c00 ? (float)x[j] : 0.f, a, r);
            // code + 128 to code: the other sign bit
            *reinterpret_cast<uint2*>(&qs[col * kRow + i % (D / 8) * 8]) =
                uint2{kv8_pack(y[0], y[1], y[2], y[3]) ^ 0x80808080u, kv8_pack(y[4], y[5], y[6], y[7]) ^ 0x80808080u};
        };
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (tid + 256 * j < cols * (D / 8)) code(tid + 256 * j, col0 ? load(tid + 256 * j + col0 * (D / 8)) : held[j]);
        __syncthreads();
        for (int ct = 0; 16 * ct < cols; ++ct) {
            int4_v acc[kWaveTiles] = {};
            // rows behind the last hold what they held: their scores are not looked at
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                const int4_v qf = *reinterpret_cast<const int4_v*>(&qs[(16 * ct + n) * kRow + 64 * k + 16 * g4]);
#pragma unroll
                for (int i = 0; i < kWaveTiles; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(m[i][k], qf, acc[i], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kWaveTiles; ++i) *reinterpret_cast<int4_v*>(&sc[16 * ct + n][16 * (kWaveTiles * wave + i) + 4 * g4]) = acc[i];
        }
        __syncthreads();
        if (nt * p.G <= kKvScoreCols) {
            for (int i = tid; i < nt * kKvScoreBlocks; i += 256) {
                const int t = i / kKvScoreBlocks, j = i % kKvScoreBlocks;
                int x = sc[t * p.G][j];
                for (int g = 1; g < p.G; ++g) x = max(x, sc[t * p.G + g][j]);
                sc[t * p.G][j] = x;
            }
        } else if (tid < kKvScoreBlocks) {  // one query: the maximum of all rounds
            for (int g = 0; g < cols; ++g) best = max(best, sc[g][tid]);
            sc[0][tid] = best;
        }
    }
    __syncthreads();
    for (int i = tid; i < nt * kKvScoreBlocks; i += 256) {
        const int t = i / kKvScoreBlocks, blk = blk0 + i % kKvScoreBlocks;
        const int pos = front + t0 + t;
        if (pos < 0 || blk >= min(pos / kKvBlock, p.nb)) continue;
        const int at = kv8_page(p.c, b, blk);
        float x = -INFINITY;  // a block without a page
        if (at >= 0) x = (float)sc[t * p.G][i % kKvScoreBlocks] * p.c.k_sum_scale[(size_t)at * p.c.Hkv + h];
        // NaN: a block that holds an infinity or NaN
        p.score[((size_t)blockIdx.y * p.T + t0 + t) * p.nb + blk] = x == x ? x : -INFINITY;
    }
}

// A score as a whole number of the same order; 0 is below every score.
__device__ __forceinline__ unsigned kv8_order(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);  // -0 ties with 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Workgroup (t, b Hkv + h): the `top` best of the row's blocks, the lowest index first among
// equals, listed ascending.  The last value that is kept is found from the top, two bits at a time,
// by counting the values that are at least as large (ballots; one barrier a round), and no further
// than where exactly `top` are.  A thread holds kN values (blocks i kThreads + thread) in registers; with
// more blocks it reads them again in each round.
template <int kThreads, int kN>
__global__ void __launch_bounds__(kThreads)
kv8_pick_kernel(Kv8SelectArgs p) {
    constexpr int kWaves = kThreads / 64, kHeld = kN * kThreads;
    __shared__ int count[3][3];  // of three rounds in turn: one's, the next one's being cleared
    __shared__ int sums[2][kWaves];
    const int b = blockIdx.y / p.c.Hkv, t = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
    const size_t row = (size_t)blockIdx.y * p.T + t;
    const float* score = p.score + row * p.nb;
    float held[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) held[j] = score[min(j * kThreads + tid, p.nb - 1)];
    const Kv8Seq sq = kv8_seq(p.c, p.len, p.n_new, b, p.T);
    if (t >= sq.n + sq.t0) return;
    if (tid < 9) count[tid / 3][tid % 3] = 0;
    const int pos = sq.len - (sq.n + sq.t0) + t;
    int* out = p.blocks + row * p.top;
    const int n = pos < 0 ? 0 : pos / kKvBlock + 1;
    for (int i = min(n, p.top) + tid; i < p.top; i += kThreads) out[i] = -1;
    if (n <= p.top) {
        for (int i = tid; i < n; i += kThreads) out[i] = i;
        return;
    }
    auto order = [&](int i, float x) {
        return i < p.first || i >= n - 1 - p.recent ? 0xffffffffu : i < p.nb ? kv8_order(x) : 0u;
    };
    unsigned u[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) u[j] = j * kThreads + tid < n ? order(j * kThreads + tid, held[j]) : 0u;
    // how many values are at least v[0], v[1], v[2] (all above 0)
    auto at_least = [&](const unsigned (&v)[3], int (&x)[3], int slot) {
        x[0] = x[1] = x[2] = 0;
        auto add = [&](unsigned y) {
#pragma unroll
            for (int k = 0; k < 3; ++k) x[k] += __popcll(__ballot(y >= v[k]));
        };
#pragma unroll
        for (int j = 0; j < kN; ++j) add(u[j]);
        for (int i0 = kHeld; i0 < n; i0 += kThreads) {
            const int i = i0 + tid;
            add(i < n ? order(i, i < p.nb ? score[i] : 0.f) : 0u);
        }
        if constexpr (kWaves > 1) {
            // a round's counts were last read two barriers before they are cleared
            if ((tid & 63) < 3) atomicAdd(&count[slot][tid & 63], (tid & 63) == 0 ? x[0] : (tid & 63) == 1 ? x[1] : x[2]);
            if (tid >= 64 && tid < 67) count[(slot + 1) % 3][tid - 64] = 0;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 3; ++k) x[k] = count[slot][k];
        }
    };
    unsigned value = 0;  // at least `top` values are at least this
    int have = n, slot = 0;
    __syncthreads();
    for (int bit = 30; bit >= 0 && have != p.top; bit -= 2, slot = (slot + 1) % 3) {
        const unsigned v[3] = {value | 1u << bit, value | 2u << bit, value | 3u << bit};
        int x[3];
        at_least(v, x, slot);
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (x[k] >= p.top) {
                value = v[k];
                have = x[k];
            }
    }
    // where more than `top` are: those above `value`, and the first of the others
    int left = n;
    if (have != p.top) {
        const unsigned v[3] = {value + 1, value + 1, value + 1};
        int x[3] = {0, 0, 0};
        if (value != 0xffffffffu) at_least(v, x, slot);
        left = p.top - x[0];
    }
    int done = 0, equal = 0;
    auto emit = [&](int i, unsigned x) {
        const bool eq = i < n && x == value;
        const unsigned long long eqs = __ballot(eq), below = (1ull << (tid & 63)) - 1;
        __syncthreads();
        if ((tid & 63) == 0) sums[0][wave] = __popcll(eqs);
        __syncthreads();
        int before = equal + __popcll(eqs & below);
        for (int w = 0; w < wave; ++w) before += sums[0][w];
        const bool take = i < n && (x > value || (eq && before < left));
        const unsigned long long takes = __ballot(take);
        if ((tid & 63) == 0) sums[1][wave] = __popcll(takes);
        __syncthreads();
        int at = done + __popcll(takes & below);
        for (int w = 0; w < wave; ++w) at += sums[1][w];
        if (take) out[at] = i;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            equal += sums[0][w];
            done += sums[1][w];
        }
    };
#pragma unroll
    for (int j = 0; j < kN; ++j)
        if (j * kThreads < n) emit(j * kThreads + tid, u[j]);
    for (int i0 = kHeld; i0 < n; i0 += kThreads) {
        const int i = i0 + tid;
        emit(i, i < n ? order(i, i < p.nb ? score[i] : 0.f) : 0u);
    }
}

inline size_t kv8_select_bytes(int B, int T, int Hkv, int nb) { return (size_t)B * Hkv * T * nb * 4; }

template <int D>
hipError_t kv8_select_d(const Kv8SelectArgs& p, hipStream_t stream) {
    const int parts = (p.nb + kKvScoreBlocks - 1) / kKvScoreBlocks;
    const dim3 grid((unsigned)((p.T + p.tq - 1) / p.tq * parts), (unsigned)(p.c.B * p.c.Hkv));
    hipLaunchKernelGGL(kv8_score_kernel<D>, grid, dim3(256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // one wave a row where its registers hold the row's scores, else 16 (32 rows of 2048 scores: 4
    // waves of 8 values a thread 11.9 us, 16 of 2 10.6)
    const dim3 rows((unsigned)p.T, (unsigned)(p.c.B * p.c.Hkv));
    if (p.nb <= 512)
        hipLaunchKernelGGL((kv8_pick_kernel<64, 8>), rows, dim3(64), 0, stream, p);
    else if (p.nb <= 2048)
        hipLaunchKernelGGL((kv8_pick_kernel<1024, 2>), rows, dim3(1024), 0, stream, p);
    else
        hipLaunchKernelGGL((kv8_pick_kernel<1024, 8>), rows, dim3(1024), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t kv8_select(const Kv8& c, const Rows16& q, const int* len, const int* n_new, int T, int Hq, int top, int first,
                      int recent, int* blocks, int nb, void* ws, hipStream_t stream) {
    const int G = Hq / c.Hkv, tq = G <= kKvScoreCols ? kKvScoreCols / G : 1;
    const Kv8SelectArgs p{c, q, len, n_new, (float*)ws, blocks, T, Hq, G, top, first, recent, nb, tq < T ? tq : T};
    if (c.D == 64) return kv8_select_d<64>(p, stream);
    if (c.D == 128) return kv8_select_d<128>(p, stream);
    return kv8_select_d<256>(p, stream);
}

size_t kv8_ws_bytes(const Kv8& c, int T, int Hq, int nb, int top) {
    const bool list = top > 0;
    const size_t part = kv8_part_bytes(c, T, Hq, kv8_plan(c, T, Hq, list ? top : nb, list));
    const size_t sel = list ? kv8_select_bytes(c.B, T, c.Hkv, nb) : 0;
    return part > sel ? part : sel;
}

}  // namespace tsa
