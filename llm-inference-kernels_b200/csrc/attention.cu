// Attention of any number of query tokens per sequence over a paged KV cache,
// on tcgen05 (fp16 operands, fp32 scores, softmax state and accumulators).
//
//   s = scale q.k             or cap tanh(scale q.k / cap), minus slope |p - j|
//   out = softmax(s) v        over the visible keys j of the query at position p
//
// One kernel serves prompts, chunks of prompts, single tokens and the two key
// sets (shared prefix, own tokens) of shared-prefix decoding.
//
// Unit: the query heads of one KV head (G of them) for up to 2 * floor(128 / G)
// consecutive tokens of one sequence; row = token * G + head. Keys are walked
// in tiles of 128 positions. The units' tiles, laid end to end, are split
// evenly over one CTA per SM, so lengths need not be known on the host and a
// few long sequences use the whole GPU; every CTA finds its share itself from
// the lengths in device memory. A unit that several CTAs share leaves
// unnormalized partial sums, joined by the second kernel in a fixed order.
//
// A CTA runs two streams (0, 1) of score tile -> softmax -> weighted sum, each
// with its own 128 softmax threads, so that one stream's matrix instructions
// run under the other's exponentials:
//   wide units (more than 128 rows): stream s holds rows [s], both read every
//     key tile;
//   paired units (up to 128 rows): both streams hold the same rows and take
//     alternate key tiles, their states are joined at the unit's end;
//   thin units (up to 16 rows, single tokens among them): paired, and with the
//     operands exchanged, scores [position][row] = K q^T and sums
//     [channel][row] = V^T w^T, so that few rows mean a small matrix product
//     instead of a padded one and a tile's softmax is one position per thread.
// Tensor memory: S0 | S1 | O0 | O1, 128 columns each. The fp16 weights overwrite
// the scores they come from and P V reads them there, with V as stored
// ([position, channel], the transposed-operand form); thin units keep them in
// shared memory.
//
// fp16 caches go from the pool to swizzled shared memory by tensor-map copies,
// one box per run of positions inside a page. INT8 caches arrive as codes and
// scales; two more warpgroups, one for K and one for V, write the codes as fp16
// integers into the same swizzled tiles, and the softmax applies the scales in
// fp32.
//
// What bounds it, measured (32 query heads on 8 KV heads; warps 0-7 softmax, 8
// copies of K and q, 9 matrix instructions, 10 schedule, 11 copies of V):
//   wide, 4096 causal tokens: a chain of latencies. 173 us in fp16 under sustained
//     load, 796 TFLOP/s, with no unit full: a tile's two steps take 4300 clocks,
//     of which the exponentials are 2048 (32768 of them, 16 per clock on an SM),
//     the tensor pipe is busy 47% of the time and the issue slots 34%. A stream's
//     next scores overwrite its weights, so their product is issued behind both
//     halves of the weighted sum, and its softmax warps wait meanwhile. Capped
//     scores 227 us, INT8 218 (scales, and one tile of K and of V in place of two);
//   thin, 16 requests of 8192: memory. 91 us in fp16, 5.9 TB/s. INT8 101 us: its
//     codes pass shared memory four times (copied in, read, written as fp16, read
//     by the matrix unit), 1500 of a tile's 3200 clocks;
//   a few tiles per CTA: the way there. 12 us for one request of 512: finding
//     the share 5000 clocks, the first copies 3000, the unit's end 2500, and the
//     joining kernel.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <mutex>

#include "lik_internal.h"
#include "lik_tcgen05.cuh"

namespace lik {

// Device error word of this file's kernels (zero when the library loads).
__device__ int g_attention_error;

namespace {

constexpr int kTile = 128;                       // key positions per tile
constexpr int kTileBytes = kTile * kHeadDim * 2; // one fp16 K or V tile
constexpr int kHalfTile = kTileBytes / 2;        // its 64-channel half
constexpr int kMaxRing = 2;                      // fp16 tiles of K, and of V, in flight
constexpr int kRaw = 2;                          // INT8 tiles of K, and of V, in flight
constexpr int kRawBytes = kTile * kHeadDim;      // codes; their scales: 256 bytes
constexpr int kScales = 4;                       // INT8: tiles whose scales are kept
constexpr int kSegs = 4;
constexpr int kThinRows = 16;
constexpr uint32_t kTmem = 0;                    // first column of tensor memory
constexpr float kLog2e = 1.4426950408889634f;
// The reference of a row's weights is put kLift powers of two below its maximum
// and raised only where a score lies more than kRaise above it, so most tiles
// leave the accumulator alone. In fp16 the weights then reach from 2^15 down: a
// row's largest is 2^7 or more, what lies 2^-21 below it and less is subnormal and
// loses 2^-32 of the largest at most (2^-25 with the reference at the maximum,
// where 32768 keys of weight 2^-25.5 vanished altogether).
constexpr float kLift = 7.0f;
constexpr float kRaise = 15.0f;
constexpr uint32_t kPolls = 1u << 18;            // a poll sleeps for a few microseconds at most

enum Mode : int { kWide = 0, kPaired = 1, kThin = 2 };
enum Dest : int { kDirect = 0, kSlot = 1, kRowBuf = 2 };
// Self test: the step whose barriers expect one arrival more than there is.
enum Stall : int {
    kNoStall, kStallQuery, kStallK, kStallV, kStallScores, kStallWeights, kStallSums, kStallSegment, kStallRaw
};

// Division of 0 <= x < 2^31 by a launch constant (the round-up method of
// Granlund and Montgomery): a multiplication instead of some thirty
// instructions, at places where the code's size counts.
struct Div {
    uint32_t d, m, s;
    __device__ __forceinline__ int operator()(int x) const {
        return static_cast<int>((__umulhi(static_cast<uint32_t>(x), m) + static_cast<uint32_t>(x)) >> s);
    }
};
Div make_div(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t{1} << s) < d) ++s;
    return {d, static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << s) - d)) / d + 1), s};
}

struct KeySet {
    const int* cu;      // [n_seq + 1] token offsets; null: token i is sequence i
    const int* ctx;     // [n_seq] live positions
    const int* tables;  // [n_seq, width]
    const int* extra;   // per token: positions that follow the keys (moves p); null: none
    int n_seq, width, n_ids, causal;
};

struct Params {
    KeySet set[2];
    int n_sets, extra_most;  // `extra` counts up to extra_most: the lengths are cut to their tables
    const int* prefix_lens;
    const int* first_keys;
    const float* slopes;
    int window;
    float kf, cap;  // scores times kf: powers of two, or tanh's argument where they are capped
    int n_tokens, n_heads, n_kv, group;
    int per, thin_per;  // tokens of 128 rows (a paired unit, half a wide one) and of a thin unit
    Div by_group, by_unit, by_block;
    int lead, weight[3];
    int num_blocks, block_size, box_rows, box_shift, total_rows;
    const __half* k_scale;
    const __half* v_scale;
    __half* out;
    int shared;      // every unit's result goes through the joining kernel
    int zero_tail;
    int slot_rows, grid;
    int stall;       // self test: the step whose wait runs out (Stall)
    float* part;     // [2 grid][slot_rows][128]
    float2* part_ml; // [2 grid][slot_rows] (maximum in powers of two, sum)
    int4* split;     // [grid] first token, tokens, head, last CTA (-1: none) of the unit split from this CTA on
    float* rowbuf;   // [2][n_tokens n_heads][128]
    float2* row_ml;
    int2* units;     // [(n_ids0 + n_ids1) n_kv] first CTA, last CTA (-1: in rowbuf)
};

struct Maps {
    CUtensorMap q[2];  // boxes of the whole tokens of 128 and of 16 rows
    CUtensorMap k, v;
};

struct Segment {
    int valid, set, seq, head;
    int tok0, ntok, mode;
    int ctx, pos0, pfx, fk;     // fk: smallest first key
    int a0, na, b0, nt;         // key tiles: na from a0, the rest from b0
    int vlo, vhi;               // positions any row sees: [fk, pfx) and [vlo, vhi]
    int t0, t1;                 // this CTA's share of the nt tiles
    int dest;
};

// A segment's list of key tiles, in registers.
struct TileList {
    int a0, na, b0;
    __device__ __forceinline__ explicit TileList(const Segment& g) : a0(g.a0), na(g.na), b0(g.b0 - g.na) {}
    __device__ __forceinline__ int operator()(int i) const { return i + (i < na ? a0 : b0); }
};

struct Misc {
    uint64_t full[2][kMaxRing], empty[2][kMaxRing], rfull[2][kRaw], rempty[2][kRaw], vscale[kScales];
    uint64_t qfull, qempty, sfull[2], pready[2][2], odone[2][2], tbar[2], segfull[kSegs], segempty[kSegs], xbar, drain;
    Segment seg[kSegs], first;
    long long scan[20];
    int heavy[20], heaviest;
    long long start, count, total;
    int start_id, start_head, start_off;
    uint32_t bad[2][kRaw];
    int low[2][2][4];  // thin units: a warp's reference is too low
    int abort;
    uint32_t tmem;
};
static_assert(sizeof(Misc) <= 2048, "the barrier block must fit behind the tiles");

struct Scales {  // INT8 caches, see convert_role
    float k[kScales][kTile], v[kScales][kTile];
    float ones[kTile / 2];
    int v_exp[kScales];
};

// Thin units, in the second query tile's place.
struct ThinRow {
    int lo, hi, fk;
    int pos;
    float slope;
};
struct ThinSpace {
    unsigned char w[2][kThinRows * 256];  // per stream: weights [2][row][64 positions], swizzled
    float l[2][kThinRows][kTile];         // each thread's part of a row's sum of weights
    float top[2][4][kThinRows], sum[2][kThinRows], ref[2][kThinRows], down[2][kThinRows], unit[2];
    uint32_t to[kThinRows];
    ThinRow row[kThinRows];
};
static_assert(sizeof(ThinSpace) <= kTileBytes, "thin space");

template <int FMT>
struct Layout {
    static constexpr int ring = FMT == kF16 ? 2 : 1;
    static constexpr int tiles = 2 * kTileBytes;  // K's, then V's
    static constexpr int v_tiles = tiles + ring * kTileBytes;
    static constexpr int raw = v_tiles + ring * kTileBytes;  // K's, then V's; then their scales
    // results on their way out, see softmax_role
    static constexpr int raw_scale = raw + 2 * kRaw * kRawBytes;
    static constexpr int stage = raw + (FMT == kF16 ? 0 : 2 * kRaw * (kRawBytes + 256));
    static constexpr int stage_bytes = FMT == kF16 ? 32768 : 16384;
    static constexpr int scales = stage + stage_bytes;
    static constexpr int misc = scales + (FMT == kF16 ? 0 : 4368);
    static_assert(sizeof(Scales) <= 4368, "scales");
    static constexpr int bytes = misc + 2048;
    static constexpr int threads = FMT == kF16 ? 384 : 640;
    // registers per thread: launched with `base`, then moved between the
    // warpgroups; the shares add up to threads * base
    static constexpr int base = FMT == kF16 ? 168 : 96;
    static constexpr int softmax_regs = FMT == kF16 ? 192 : 136;
    static constexpr int other_regs = FMT == kF16 ? 120 : 80;
    static constexpr int convert_regs = 64;
    static_assert(2 * softmax_regs + other_regs + (FMT == kF16 ? 0 : 2 * convert_regs) <= threads / 128 * base,
                  "register shares exceed what the block is launched with");
};

template <int N>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ---- bounded waits -----------------------------------------------------------

// Whole warp; every lane has observed the phase on return. False: give up
// (this wait or another one of the CTA ran out; the kernel's end reports it).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Misc* m, uint32_t polls = kPolls) {
#pragma unroll 1
    for (uint32_t i = 0;; ++i) {
        if (__all_sync(kFull, mbar_try_wait(bar, parity))) return true;
        if (i == polls) *reinterpret_cast<volatile int*>(&m->abort) = 1;
        if (*reinterpret_cast<volatile int*>(&m->abort)) return false;
    }
}
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// ---- units -------------------------------------------------------------------

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ int cu_at(const KeySet& k, int b, int n_tokens) {
    return k.cu ? clampi(k.cu[b], 0, n_tokens) : b;
}

// Unit numbers of a key set: b is the first unit of sequence b; the others of a
// sequence whose tokens start at c are n_seq + c / unit and following (some
// numbers are nobody's). The sequence that a number from n_seq on belongs to:
__device__ __forceinline__ int seq_of(const KeySet& k, int extra, Div by_unit, int n_tokens) {
    int lo = 0, hi = k.n_seq - 1;  // largest b with cu[b] / unit <= extra
#pragma unroll 1
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (by_unit(cu_at(k, mid, n_tokens)) <= extra) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Fills the unit `id` (all heads alike); false if no tokens carry this number.
__device__ bool make_unit(const Params& p, int id, Segment& s) {
    s.set = id < p.set[0].n_ids ? 0 : 1;
    const KeySet& k = p.set[s.set];
    if (s.set) id -= p.set[0].n_ids;
    if (k.n_seq <= 0) return false;
    const int unit = 2 * p.per;
    const int b = id < k.n_seq ? id : seq_of(k, id - k.n_seq, p.by_unit, p.n_tokens);
    const int c0 = cu_at(k, b, p.n_tokens);
    const int n = k.cu ? cu_at(k, b + 1, p.n_tokens) - c0 : 1;
    const int at = id < k.n_seq ? 0 : (id - k.n_seq - p.by_unit(c0) + 1) * unit;
    if (at < 0 || at >= n || (id >= k.n_seq && at == 0)) return false;
    s.seq = b;
    s.tok0 = c0 + at;
    s.ntok = min(unit, n - at);
    s.mode = s.ntok <= p.thin_per ? kThin : s.ntok <= p.per ? kPaired : kWide;
    s.ctx = static_cast<int>(min(static_cast<long long>(max(k.ctx[b], 0)),
                                 static_cast<long long>(k.width) * p.block_size));
    s.pos0 = s.ctx - n + at;
    s.pfx = p.prefix_lens && s.set == 0 ? clampi(p.prefix_lens[b], 0, s.ctx) : 0;
    const int fk = p.first_keys ? max(p.first_keys[s.tok0], 0) : 0;  // they do not decrease
    s.fk = fk;
    s.vlo = p.window > 0 ? max(s.pos0 - p.window + 1, fk) : fk;
    s.vhi = k.causal ? min(s.pos0 + s.ntok - 1, s.ctx - 1) : s.ctx - 1;
    s.a0 = s.na = s.b0 = 0;
    if (s.pfx > fk) {
        s.a0 = fk / kTile;
        s.na = (s.pfx - 1) / kTile - s.a0 + 1;
    }
    s.nt = s.na;
    if (s.vhi >= s.vlo) {
        s.b0 = max(s.vlo / kTile, s.a0 + s.na);
        s.nt += max(s.vhi / kTile - s.b0 + 1, 0);
    }
    return true;
}

// ---- softmax of one stream -----------------------------------------------------

struct Row {  // what one softmax thread's row sees
    int lo, hi, fk, pfx, pos;
    float slope;
};

// 1 / a row's sum of weights: 0 where it saw nothing; what is not finite stays so.
__device__ __forceinline__ float over_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }

// tanh on [-0.7, 0.7] as an odd polynomial of degree 9 with linear coefficient 1,
// minimax in the relative error (3.5e-7): Remez exchange on tanh(t) / t over t^2.
// A capped score is so within a few fp32 roundings of its own, however loose the cap.
constexpr float kTanhNear = 0.7f;
constexpr float kTanh3 = -0.33331084995633364f, kTanh5 = 0.13287660176553176f, kTanh7 = -0.05101637469806898f,
                kTanh9 = 0.013938170996101448f;
struct TanhNear {  // up tanh(t) for |t| <= 0.7
    float2 c[5];
    __device__ __forceinline__ explicit TanhNear(float up) {
        const float k[5] = {1.0f, kTanh3, kTanh5, kTanh7, kTanh9};
#pragma unroll
        for (int i = 0; i < 5; ++i) c[i] = {k[i] * up, k[i] * up};
    }
    __device__ __forceinline__ float2 operator()(float2 t) const {
        const float2 y = mul2(t, t);
        return mul2(fma2(fma2(fma2(fma2(c[4], y, c[3]), y, c[2]), y, c[1]), y, c[0]), t);
    }
};
// tanh of any t: the polynomial, or 1 - 2 / (1 + e^2t), which cancels near zero
__device__ __forceinline__ float tanh_any(float t) {
    const float y = t * t;
    const float near = t * fmaf(fmaf(fmaf(fmaf(kTanh9, y, kTanh7), y, kTanh5), y, kTanh3), y, 1.0f);
    const float far = 1.0f - 2.0f * fast_rcp(1.0f + fast_exp2(t * (2.0f * kLog2e)));
    return fabsf(t) <= kTanhNear ? near : far;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float d;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// A load from shared memory that stays where it is written (lifted out of the
// loop below, a step's scales alone would fill the registers).
__device__ __forceinline__ float4 load_scales(const float4* p) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_addr(p)));
    return v;
}
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {  // bits lo .. hi of a word
    const uint32_t from = lo <= 0 ? ~0u : lo > 31 ? 0u : ~0u << lo;
    const uint32_t to = hi >= 31 ? ~0u : hi < 0 ? 0u : (2u << hi) - 1u;
    return from & to;
}

// W scores that are not all near zero, capped in place: up tanh(k s), 16 columns at
// a time (rolled: this code beside the step's own would crowd the instruction
// cache, and capped scores are mostly near).
template <int W, bool I8>
__device__ __forceinline__ void cap_far(float up, float kf, uint32_t s_addr, const float4* ks) {
#pragma unroll 1
    for (int i0 = 0; i0 < W; i0 += 16) {
        float s[16];
        tmem_ld16(s_addr + i0, s);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 k = I8 ? load_scales(ks + (i0 + i) / 4) : float4{kf, kf, kf, kf};
            s[i] = up * tanh_any(s[i] * k.x);
            s[i + 1] = up * tanh_any(s[i + 1] * k.y);
            s[i + 2] = up * tanh_any(s[i + 2] * k.z);
            s[i + 3] = up * tanh_any(s[i + 3] * k.w);
        }
        tmem_st16(s_addr + i0, reinterpret_cast<const uint32_t*>(s));
    }
    tmem_wait_st();
}

// One step: the softmax of W score columns at s_addr, keys from j0, into W fp16
// weights at p_addr. `m` is the row's reference, in powers of two. The weights
// are worked out with the reference so far; only where a score turns out to lie
// more than 2^kRaise above it (in the first step of a unit, rarely later) the
// maximum is searched for, the reference raised and the weights worked out
// again. Searched for ahead of the weights it held up every step by a quarter.
// Weights stay below 2^15, which fp16 holds.
//
// INT8: ks holds kf times K's scales, vs V's scales divided by 2^v_exp, the
// largest so far; the sums are in units of 2^ev. The matrix instructions see the
// exact codes. Scales may have any sign or be no number: they are applied before
// a key is hidden, and `ones` stands in for them afterwards.
template <int W, bool I8, bool MOD>
__device__ __forceinline__ bool softmax_step(const Params& p, Misc* mi, const Row& row, uint32_t s_addr, uint32_t p_addr,
                                             uint32_t o_addr, int j0, bool have_sums, uint64_t* odone, uint32_t odone_parity,
                                             const float4* ks, const float4* vs, const float4* ones, int v_exp, float& m,
                                             float& l, int& ev) {
    float s[W];
#pragma unroll
    for (int i = 0; i < W; i += 32) tmem_ld32(s_addr + i, s + i);
    tmem_wait_ld();
    if (MOD) {  // scores to powers of two, or tanh's arguments
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const float4 k = I8 ? load_scales(ks + i / 4) : float4{p.kf, p.kf, p.kf, p.kf};
            const float2 a = mul2({s[i], s[i + 1]}, {k.x, k.y}), b = mul2({s[i + 2], s[i + 3]}, {k.z, k.w});
            s[i] = a.x;
            s[i + 1] = a.y;
            s[i + 2] = b.x;
            s[i + 3] = b.y;
        }
        if (p.cap > 0.f) {
            const float up = p.cap * kLog2e;
            float far[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < W; i += 2) far[i / 2 & 3] = max3_abs(far[i / 2 & 3], s[i], s[i + 1]);
            if (__all_sync(kFull, fmaxf(max3(far[0], far[1], far[2]), far[3]) <= kTanhNear)) {
                const TanhNear near(up);
#pragma unroll
                for (int i = 0; i < W; i += 2) {
                    const float2 t = near({s[i], s[i + 1]});
                    s[i] = t.x;
                    s[i + 1] = t.y;
                }
            } else {
                cap_far<W, I8>(up, p.kf, s_addr, ks);
#pragma unroll
                for (int i = 0; i < W; i += 32) tmem_ld32(s_addr + i, s + i);
                tmem_wait_ld();
            }
        }
        if (p.slopes) {
            const float from = static_cast<float>(j0 - row.pos);
#pragma unroll
            for (int i = 0; i < W; ++i) s[i] = fmaf(-row.slope, fabsf(from + static_cast<float>(i)), s[i]);
        }
    }
    const bool whole = (j0 >= row.lo && j0 + W - 1 <= row.hi) || (j0 >= row.fk && j0 + W <= row.pfx);
    if (__any_sync(kFull, !whole)) {
        if (I8 && !MOD) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const float4 k = load_scales(ks + i / 4);
                s[i] *= k.x;
                s[i + 1] *= k.y;
                s[i + 2] *= k.z;
                s[i + 3] *= k.w;
            }
            ks = ones;
        }
#pragma unroll
        for (int i = 0; i < W; i += 32) {
            const int j = j0 + i;
            const uint32_t see = bits_between(row.lo - j, row.hi - j) | bits_between(row.fk - j, row.pfx - 1 - j);
#pragma unroll
            for (int c = 0; c < 32; ++c) s[i + c] = (see >> c) & 1u ? s[i + c] : -INFINITY;
        }
    }
    const float kf = MOD ? 1.f : p.kf;
#pragma unroll 1
    for (bool again = false;; again = true) {
        const float ms = m == -INFINITY ? 0.f : -m;
        const float2 ms2 = {ms, ms};
        float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
        float over[2] = {-INFINITY, -INFINITY};
        uint32_t w[16];
        float4 k4{}, v4{};
#pragma unroll
        for (int c = 0; c < W / 2; ++c) {
            const float a = s[2 * c], b = s[2 * c + 1];
            float2 k = {kf, kf}, v = {1.f, 1.f};
            if (I8) {
                if (c % 2 == 0) {
                    k4 = MOD ? float4{1.f, 1.f, 1.f, 1.f} : load_scales(ks + c / 2);
                    v4 = load_scales(vs + c / 2);
                }
                k = c & 1 ? float2{k4.z, k4.w} : float2{k4.x, k4.y};
                v = c & 1 ? float2{v4.z, v4.w} : float2{v4.x, v4.y};
            }
            float2 x = MOD ? add2({a, b}, ms2) : fma2({a, b}, k, ms2);
            over[c & 1] = max3(over[c & 1], x.x, x.y);
            x.x = fast_exp2(x.x);
            x.y = fast_exp2(x.y);
            sum[c & 1] = add2(sum[c & 1], x);
            if (I8) x = mul2(x, v);
            w[c % 16] = pack_f16(x.x, x.y);
            if (c % 16 == 15) tmem_st16(p_addr + c - 15, w);
        }
        const bool low = fmaxf(over[0], over[1]) > kRaise || m == -INFINITY;
        if (again || !__any_sync(kFull, low || (I8 && v_exp > ev))) {
            const float2 all = add2(sum[0], sum[1]);
            l += all.x + all.y;
            return true;
        }
        tmem_wait_st();
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const float4 k = I8 && !MOD ? load_scales(ks + i / 4) : float4{kf, kf, kf, kf};
            top = max3(top, s[i] * k.x, s[i + 1] * k.y);
            top = max3(top, s[i + 2] * k.z, s[i + 3] * k.w);
        }
        const float up = fmaxf(m, top - kLift);
        const float f = m == -INFINITY ? 0.f : fast_exp2(m - up);
        m = up;
        l *= f;
        float fo = f;
        if (I8) {
            fo *= fast_exp2(static_cast<float>(ev - v_exp));
            ev = v_exp;
        }
        if (have_sums) {
            if (odone && !warp_wait(odone, odone_parity, mi)) return false;
            tcgen05_fence_after();
#pragma unroll 1
            for (int c = 0; c < kHeadDim; c += 16) {
                float o[16];
                tmem_ld16(o_addr + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] *= fo;
                tmem_st16(o_addr + c, reinterpret_cast<const uint32_t*>(o));
            }
        }
    }
}

// All of a stream's tiles of a wide or paired segment, each in two steps of 64
// columns, the first one's weights being multiplied with V while the second is
// worked out. A tile's scores are there only after the products of the tile
// before, so the sums can be scaled at once in a tile's first step and after the
// first half's product in its second. `tiles` and `halves` count the tiles so
// far (of all segments, of these ones), `before` those of earlier segments.
template <bool I8, bool MOD>
__device__ __forceinline__ bool softmax_run(const Params& p, Misc* mi, const Scales* scales, const Segment& g,
                                            const Row& row, int stream, uint32_t before, uint32_t s_addr,
                                            uint32_t o_addr, uint32_t& tiles, uint32_t& halves, float& m, float& l,
                                            int& ev) {
    constexpr int W = 64;
    const int step = g.mode == kWide ? 1 : 2;
    const int t0 = g.t0, t1 = g.t1, i0 = t0 + (g.mode == kWide ? 0 : stream);
    const TileList tile(g);
#pragma unroll 1
    for (int i = i0; i < t1; i += step) {
        if (!warp_wait(&mi->sfull[stream], tiles & 1, mi)) return false;
        ++tiles;
        tcgen05_fence_after();
        const int j0 = tile(i) * kTile;
        const uint32_t at = before + i - t0, st = at % kScales;
        if (I8 && !warp_wait(&mi->vscale[st], (at / kScales) & 1, mi)) return false;
        const int v_exp = I8 ? scales->v_exp[st] : 0;
#pragma unroll 1
        for (int c = 0; c < kTile; c += W) {
            const float4* ks = reinterpret_cast<const float4*>(scales->k[st] + c);
            if (!softmax_step<W, I8, MOD>(p, mi, row, s_addr + c, s_addr + c / 2, o_addr, j0 + c, i > i0 || c > 0,
                                     c > 0 ? &mi->odone[stream][0] : nullptr, halves & 1, ks,
                                     reinterpret_cast<const float4*>(scales->v[st] + c),
                                     reinterpret_cast<const float4*>(scales->ones), v_exp, m, l, ev))
                return false;
            tmem_wait_st();
            tcgen05_fence_before();
            warp_arrive(&mi->pready[stream][c > 0]);
        }
        ++halves;
    }
    return true;
}

// Where row (tok, query head hr) of the segment goes: a row of out, of the
// CTA's partial sums (`ur` its row in the unit) or of the whole units' sums.
__device__ __forceinline__ uint32_t dest_row(const Params& p, const Segment& g, int tok, int hr, int ur) {
    const uint32_t r = static_cast<uint32_t>(tok) * p.n_heads + hr;
    if (g.dest == kDirect) return r;
    if (g.dest == kSlot) return (2 * blockIdx.x + (g.t0 == 0)) * p.slot_rows + ur;
    return static_cast<uint32_t>(g.set) * p.n_tokens * p.n_heads + r;
}
__device__ __forceinline__ void store_ml(const Params& p, const Segment& g, uint32_t row, float m, float l) {
    if (g.dest != kDirect) (g.dest == kSlot ? p.part_ml : p.row_ml)[row] = {m, l};
}

// Barrier of the eight softmax warps.
__device__ __forceinline__ bool softmax_sync(Misc* mi, uint32_t& phase) {
    warp_arrive(&mi->xbar);
    return warp_wait(&mi->xbar, phase++ & 1, mi);
}

// Writes this warp's 32 rows of a stream's sums, times `f`, as fp16 or fp32
// rows of 128 channels; `row_at` is this lane's row, ~0 for none.
template <int FMT, bool HALF>
__device__ __forceinline__ void store_wide(unsigned char* stage, unsigned char* base, uint32_t o_addr, bool any,
                                           uint32_t row_at, float f) {
    constexpr int bytes = Layout<FMT>::stage_bytes / 256;  // of a row per pass
    constexpr int lanes = bytes / 16, cols = HALF ? bytes / 2 : bytes / 4;
    const int lane = threadIdx.x & 31;
    unsigned char* const mine = stage + (threadIdx.x >> 5) * 32 * bytes;
#pragma unroll 1
    for (int c = 0; c < kHeadDim; c += cols) {
        float o[cols];
#pragma unroll
        for (int i = 0; i < cols; ++i) o[i] = 0.f;
        if (any) {
            if constexpr (cols == 16) {
                tmem_ld16(o_addr + c, o);
            } else {
#pragma unroll
                for (int i = 0; i < cols; i += 32) tmem_ld32(o_addr + c + i, o + i);
            }
            tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < lanes; ++i) {
            uint4 u;
            if constexpr (HALF) {
                u = {pack_f16(o[8 * i] * f, o[8 * i + 1] * f), pack_f16(o[8 * i + 2] * f, o[8 * i + 3] * f),
                     pack_f16(o[8 * i + 4] * f, o[8 * i + 5] * f), pack_f16(o[8 * i + 6] * f, o[8 * i + 7] * f)};
            } else {
                u = {__float_as_uint(o[4 * i] * f), __float_as_uint(o[4 * i + 1] * f),
                     __float_as_uint(o[4 * i + 2] * f), __float_as_uint(o[4 * i + 3] * f)};
            }
            *reinterpret_cast<uint4*>(mine + lane * bytes + ((i ^ (lane & (lanes - 1))) << 4)) = u;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < lanes; ++i) {
            const int r = i * (32 / lanes) + lane / lanes, x = lane & (lanes - 1);
            const uint32_t at = __shfl_sync(kFull, row_at, r);
            const uint4 u = *reinterpret_cast<const uint4*>(mine + r * bytes + ((x ^ (r & (lanes - 1))) << 4));
            if (at != ~0u)
                *reinterpret_cast<uint4*>(base + (static_cast<size_t>(at) * kHeadDim + c) * (HALF ? 2 : 4) + x * 16) = u;
        }
        __syncwarp();
    }
}

// Barrier of a stream's four softmax warps.
__device__ __forceinline__ bool stream_sync(Misc* mi, int stream, uint32_t& phase) {
    warp_arrive(&mi->tbar[stream]);
    return warp_wait(&mi->tbar[stream], phase++ & 1, mi);
}

// A thin segment. Scores come transposed, [position][row], so a thread holds one
// position's scores of all rows; a row's reference is the same in all 128
// threads of the stream, and each keeps its own part of the sum of weights. A
// vote per tile finds out whether any reference has to be raised first. Four
// rows at a time, in loops: unrolled over the rows the kernel was twice as large
// and waited for its instructions.
template <int FMT, bool MOD>
__device__ bool thin_segment(const Params& p, Misc* mi, unsigned char* smem, const Segment& g, int stream, uint32_t before,
                             uint32_t s_addr, uint32_t o_addr, uint32_t& tiles, uint32_t& tphase, uint32_t& votes,
                             uint32_t& xphase, bool wide_before) {
    constexpr bool I8 = FMT != kF16;
    constexpr int NT = kThinRows;
    const int r_in = threadIdx.x & 127, lane = threadIdx.x & 31, warp = r_in >> 5;
    ThinSpace* const sp = reinterpret_cast<ThinSpace*>(smem + kTileBytes);
    const Scales* scales = reinterpret_cast<const Scales*>(smem + Layout<FMT>::scales);
    const KeySet& ks = p.set[g.set];
    const int rows = g.ntok * p.group, pfx = g.pfx;
    if (r_in < NT) {  // both streams write the same
        const int tl = p.by_group(r_in), tok = g.tok0 + tl;
        ThinRow q = {0, -1, 0, 0, 0.f};
        if (r_in < rows) {
            const int pos = ks.extra ? clampi(ks.extra[tok], 0, p.extra_most) + g.ctx - 1 : g.pos0 + tl;
            q.fk = p.first_keys ? max(p.first_keys[tok], 0) : 0;
            q.lo = max(p.window > 0 ? max(pos - p.window + 1, 0) : 0, q.fk);
            q.hi = ks.causal ? min(pos, g.ctx - 1) : g.ctx - 1;
            q.pos = pos;
            if (MOD && p.slopes) q.slope = p.slopes[g.head * p.group + r_in - tl * p.group] * kLog2e;
        }
        sp->row[r_in] = q;
        sp->ref[stream][r_in] = -INFINITY;
    }
    if (!stream_sync(mi, stream, tphase)) return false;
    int lo_max = 0, hi_min = 0x7fffffff, fk_max = 0;
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
        lo_max = max(lo_max, sp->row[r].lo);
        hi_min = min(hi_min, sp->row[r].hi);
        fk_max = max(fk_max, sp->row[r].fk);
    }
    float* const ref = sp->ref[stream];
    float* const l = &sp->l[stream][0][r_in];
    const int rows4 = (rows + 3) & ~3;
#pragma unroll 1
    for (int r = 0; r < rows4; ++r) l[r * kTile] = 0.f;
    int ev = -200;
    const int t0 = g.t0, t1 = g.t1;
    const TileList tile(g);
    unsigned char* const w_at = sp->w[stream] + (r_in >> 6) * (kThinRows * 128) + (r_in & 7) * 2;
    const int chunk = (r_in & 63) >> 3;
    bool any = false;
#pragma unroll 1
    for (int i = t0 + stream; i < t1; i += 2, any = true) {
        const int j0 = tile(i) * kTile, j = j0 + r_in;
        if (!warp_wait(&mi->sfull[stream], tiles & 1, mi)) return false;
        ++tiles;
        tcgen05_fence_after();
        const uint32_t at = before + i - t0, st = at % kScales;
        if (I8 && !warp_wait(&mi->vscale[st], (at / kScales) & 1, mi)) return false;
        const int v_exp = I8 ? scales->v_exp[st] : 0;
        const float vx = I8 ? scales->v[st][r_in] : 1.f;
        const float kx = I8 ? scales->k[st][r_in] : p.kf;
        const bool whole = (j0 >= lo_max && j0 + kTile - 1 <= hi_min) || (j0 >= fk_max && j0 + kTile <= pfx);
        bool low = I8 && v_exp > ev;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 4) {  // scores in powers of two, -inf where hidden, written back
            float x[4];
            tmem_ld4(s_addr + r0, x);
            const float4 m4 = *reinterpret_cast<const float4*>(ref + r0);
            const float m[4] = {m4.x, m4.y, m4.z, m4.w};
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                x[c] *= kx;
                if (MOD && p.cap > 0.f) x[c] = p.cap * kLog2e * tanh_any(x[c]);
                if (MOD && p.slopes)
                    x[c] = fmaf(-sp->row[r0 + c].slope, fabsf(static_cast<float>(j - sp->row[r0 + c].pos)), x[c]);
                if (!whole || r0 + c >= rows) {
                    const ThinRow& q = sp->row[r0 + c];
                    if (!((j >= q.lo && j <= q.hi) || (j >= q.fk && j < pfx && r0 + c < rows))) x[c] = -INFINITY;
                }
                low = low || x[c] - m[c] > kRaise;
            }
            tmem_st4(s_addr + r0, x);
        }
        tmem_wait_st();
        low = __any_sync(kFull, low);
        int* const flag = mi->low[stream][votes++ & 1];
        if (lane == 0) *reinterpret_cast<volatile int*>(flag + warp) = low;
        if (!stream_sync(mi, stream, tphase)) return false;
        const volatile int* f = flag;
        if (f[0] | f[1] | f[2] | f[3]) {  // raise the references by the tile's maxima
#pragma unroll 1
            for (int r0 = 0; r0 < rows; r0 += 4) {
                float x[4];
                tmem_ld4(s_addr + r0, x);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int d = 16; d; d >>= 1) x[c] = fmaxf(x[c], __shfl_xor_sync(kFull, x[c], d));
                    if (lane == 0) sp->top[stream][warp][r0 + c] = x[c];
                }
            }
            if (!stream_sync(mi, stream, tphase)) return false;
            if (r_in < rows) {
                const float old = ref[r_in];
                const float top = fmaxf(fmaxf(sp->top[stream][0][r_in], sp->top[stream][1][r_in]),
                                        fmaxf(sp->top[stream][2][r_in], sp->top[stream][3][r_in]));
                const float up = fmaxf(old, top - kLift);
                sp->down[stream][r_in] = old == -INFINITY ? 0.f : fast_exp2(old - up);
                ref[r_in] = up;
            }
            if (!stream_sync(mi, stream, tphase)) return false;
            float fo = 1.f;
            if (I8) {
                fo = fast_exp2(static_cast<float>(ev - v_exp));
                ev = v_exp;
            }
            if (any) {  // this stream's products so far are done: the scores came after them
#pragma unroll 1
                for (int r0 = 0; r0 < rows; r0 += 4) {
                    float x[4];
                    tmem_ld4(o_addr + r0, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float d = r0 + c < rows ? sp->down[stream][r0 + c] : 0.f;
                        l[(r0 + c) * kTile] *= d;
                        x[c] *= d * fo;
                    }
                    tmem_st4(o_addr + r0, x);
                }
                tmem_wait_st();
            }
        }
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 4) {
            float x[4];
            tmem_ld4(s_addr + r0, x);
            const float4 m4 = *reinterpret_cast<const float4*>(ref + r0);
            const float m[4] = {m4.x, m4.y, m4.z, m4.w};
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = r0 + c;
                const float e = fast_exp2(x[c] - (m[c] == -INFINITY ? 0.f : m[c]));
                l[r * kTile] += e;
                *reinterpret_cast<__half*>(w_at + r * 128 + ((chunk ^ (r & 7)) << 4)) = __float2half_rn(e * vx);
            }
        }
        fence_async_smem();  // the weights, for the matrix instructions
        tcgen05_fence_before();
        warp_arrive(&mi->pready[stream][1]);
    }
    if (any) {
        if (!warp_wait(&mi->odone[stream][1], (tiles - 1) & 1, mi)) return false;
        tcgen05_fence_after();
    }
    if (wide_before && !softmax_sync(mi, xphase)) return false;  // the staging space was the warps' own
    // Join the two streams; a thread holds one channel of all rows now. Stream
    // 1 hands its sums over, stream 0 scales both to a row's common reference.
    float* const other = reinterpret_cast<float*>(smem + Layout<FMT>::stage) + r_in;  // [row][channel]
    if (stream == 1) {
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 4) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (any) {
                tmem_ld4(o_addr + r0, x);
                tmem_wait_ld();
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) other[(r0 + c) * kHeadDim] = x[c];
        }
    }
    if (!stream_sync(mi, stream, tphase)) return false;
#pragma unroll 1
    for (int r = warp; r < rows; r += 4) {
        const float4 q = *reinterpret_cast<const float4*>(&sp->l[stream][r][lane * 4]);
        float t = (q.x + q.y) + (q.z + q.w);
#pragma unroll
        for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(kFull, t, d);
        if (lane == 0) sp->sum[stream][r] = t;
    }
    if (r_in == 0) sp->unit[stream] = I8 && any ? fast_exp2(static_cast<float>(ev)) : 1.f;
    if (!softmax_sync(mi, xphase)) return false;
    if (stream == 0) {
        if (r_in < rows) {
            const float m0 = sp->ref[0][r_in], m1 = sp->ref[1][r_in], top = fmaxf(m0, m1);
            const float a0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - top), a1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - top);
            const float sum = a0 * sp->sum[0][r_in] + a1 * sp->sum[1][r_in];
            const int tl = p.by_group(r_in);
            const uint32_t to = dest_row(p, g, g.tok0 + tl, g.head * p.group + r_in - tl * p.group, r_in);
            store_ml(p, g, to, top, sum);
            const float inv = g.dest != kDirect ? 1.f : over_sum(sum);
            sp->down[0][r_in] = a0 * sp->unit[0] * inv;
            sp->down[1][r_in] = a1 * sp->unit[1] * inv;
            sp->to[r_in] = to;
        }
        if (!stream_sync(mi, stream, tphase)) return false;
        const int dest = g.dest;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 4) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (any) {
                tmem_ld4(o_addr + r0, x);
                tmem_wait_ld();
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = r0 + c;
                if (r >= rows) break;
                const float f0 = sp->down[0][r], f1 = sp->down[1][r];
                const float v = (f0 != 0.f ? x[c] * f0 : 0.f) + (f1 != 0.f ? other[r * kHeadDim] * f1 : 0.f);
                const size_t e = static_cast<size_t>(sp->to[r]) * kHeadDim + r_in;
                if (dest == kDirect)
                    p.out[e] = __float2half_rn(v);
                else
                    (dest == kSlot ? p.part : p.rowbuf)[e] = v;
            }
        }
    }
    fence_async_smem();  // queries may be copied over the space that was used here
    if (!softmax_sync(mi, xphase)) return false;
    tcgen05_fence_before();
    return true;
}

// Results leave through shared memory, so that a warp writes whole runs of a
// row instead of 16 bytes of 32 rows (a quarter of the time for a wide unit).
template <int FMT, bool MOD>
__device__ void softmax_role(const Params& p, Misc* mi, unsigned char* smem) {
    const int stream = threadIdx.x >> 7, r_in = threadIdx.x & 127;
    const uint32_t lane_base = static_cast<uint32_t>(r_in & 96) << 16;
    const uint32_t s_addr = kTmem + lane_base + stream * 128, o_addr = s_addr + 256;
    unsigned char* const stage = smem + Layout<FMT>::stage;
    const Scales* scales = reinterpret_cast<const Scales*>(smem + Layout<FMT>::scales);
    constexpr bool I8 = FMT != kF16;
    uint32_t tiles = 0, halves = 0, before = 0, xphase = 0, tphase = 0, votes = 0;
    bool wide_before = false;
    for (uint32_t k = 0;; ++k) {
        const int slot = k % kSegs;
        if (!warp_wait(&mi->segfull[slot], (k / kSegs) & 1, mi)) return;
        const Segment& g = mi->seg[slot];
        if (!g.valid) return;
        if (g.mode == kThin) {
            const uint32_t b = before;
            before += g.t1 - g.t0;
            const bool ok =
                thin_segment<FMT, MOD>(p, mi, smem, g, stream, b, s_addr, o_addr, tiles, tphase, votes, xphase,
                                          wide_before);
            if (!ok) return;
            wide_before = false;
            warp_arrive(&mi->segempty[slot]);
            continue;
        }
        const KeySet& ks = p.set[g.set];
        const bool wide = g.mode == kWide;
        const int tl0 = p.by_group(r_in), hr = g.head * p.group + r_in - tl0 * p.group;
        const int tl = tl0 + (wide ? stream * p.per : 0);
        const bool live = tl < g.ntok && tl0 < p.per;
        const int tok = g.tok0 + tl;
        Row row{0, 0x7fffffff, 0, 0, 0, 0.f};  // a row that is not live keeps every column: nothing reads it
        if (live) {
            const int pos = ks.extra ? clampi(ks.extra[tok], 0, p.extra_most) + g.ctx - 1 : g.pos0 + tl;
            row.fk = p.first_keys ? max(p.first_keys[tok], 0) : 0;
            row.lo = max(p.window > 0 ? max(pos - p.window + 1, 0) : 0, row.fk);
            row.hi = ks.causal ? min(pos, g.ctx - 1) : g.ctx - 1;
            row.pfx = g.pfx;
            row.pos = pos;
            if (MOD && p.slopes) row.slope = p.slopes[hr] * kLog2e;
        }
        float m = -INFINITY, l = 0.f;
        int ev = -200;
        const int mine = wide ? g.t1 - g.t0 : (g.t1 - g.t0 - stream + 1) / 2;  // tiles of this stream
        if (!softmax_run<I8, MOD>(p, mi, scales, g, row, stream, before, s_addr, o_addr, tiles, halves, m, l, ev)) return;
        before += g.t1 - g.t0;
        const float unit_v = I8 && mine > 0 ? fast_exp2(static_cast<float>(ev)) : 1.f;
        if (mine > 0) {
            if (!warp_wait(&mi->odone[stream][1], (tiles - 1) & 1, mi)) return;
            tcgen05_fence_after();
        }
        // l is 0 for a row that saw nothing, NaN if a score was
        const float m2 = l == 0.f ? -INFINITY : fmaxf(m, -FLT_MAX);
        if (wide) {
            const uint32_t row_at = live ? dest_row(p, g, tok, hr, tl * p.group + hr - g.head * p.group) : ~0u;
            if (live) store_ml(p, g, row_at, m2, l);
            if (g.dest == kDirect)
                store_wide<FMT, true>(stage, reinterpret_cast<unsigned char*>(p.out), o_addr, mine > 0, row_at,
                                      unit_v * over_sum(l));
            else
                store_wide<FMT, false>(stage, reinterpret_cast<unsigned char*>(g.dest == kSlot ? p.part : p.rowbuf),
                                       o_addr, mine > 0, row_at, unit_v);
        } else {
            // join the streams: each scales its sums to the row's common
            // reference, then 256 threads add the two in order
            if (wide_before && !softmax_sync(mi, xphase)) return;  // the staging space was the warps' own
            float2* ml = reinterpret_cast<float2*>(stage);
            float4* data = reinterpret_cast<float4*>(stage + 2048);
            const int rows = g.ntok * p.group;
            ml[threadIdx.x] = live ? float2{m2, l} : float2{-INFINITY, 0.f};
            if (!softmax_sync(mi, xphase)) return;
            const float top = fmaxf(ml[r_in].x, ml[kTile + r_in].x);
            const float f = m2 == -INFINITY ? 0.f : fast_exp2(m2 - top) * unit_v;
            int dc = 128;  // channels per pass: what fits the scratch space (2 * rows <= 256)
            while (2 * rows * dc * 4 > Layout<FMT>::stage_bytes - 2048) dc >>= 1;
            const int quads = dc / 4, spread = min(quads, 8) - 1;
            float4* const mine_at = data + (stream * rows + r_in) * quads;
#pragma unroll 1
            for (int d0 = 0; d0 < kHeadDim; d0 += dc) {
#pragma unroll 1
                for (int c = 0; c < dc; c += 32) {
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                    if (mine > 0) {
                        tmem_ld32(o_addr + ((d0 + c) & ~31), o);
                        tmem_wait_ld();
                    }
                    if (live) {
                        const int skip = ((d0 + c) & 31) / 4, n = min(quads, 8);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int x = i - skip;
                            if (x >= 0 && x < n) {
                                float4 v = {o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f, o[4 * i + 3] * f};
                                if (f == 0.f) v = {0.f, 0.f, 0.f, 0.f};
                                mine_at[(c / 4 + x) ^ (r_in & spread)] = v;
                            }
                        }
                    }
                }
                if (!softmax_sync(mi, xphase)) return;
#pragma unroll 1
                for (int it = threadIdx.x; it < rows * quads; it += 256) {
                    const int r = it / quads, c4 = it - r * quads;
                    const float2 e0 = ml[r], e1 = ml[kTile + r];
                    const float mx = fmaxf(e0.x, e1.x);
                    const float sum = (e0.x > -INFINITY ? e0.y * fast_exp2(e0.x - mx) : 0.f) +
                                      (e1.x > -INFINITY ? e1.y * fast_exp2(e1.x - mx) : 0.f);
                    const float4 a = data[r * quads + (c4 ^ (r & spread))], b = data[(rows + r) * quads + (c4 ^ (r & spread))];
                    const float4 v = {a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w};
                    const int tk = p.by_group(r);
                    const uint32_t at = dest_row(p, g, g.tok0 + tk, g.head * p.group + r - tk * p.group, r);
                    if (d0 == 0 && c4 == 0) store_ml(p, g, at, mx, sum);
                    const size_t e = static_cast<size_t>(at) * kHeadDim + d0 + 4 * c4;
                    if (g.dest == kDirect) {
                        const float inv = over_sum(sum);
                        *reinterpret_cast<uint2*>(p.out + e) = {pack_f16(v.x * inv, v.y * inv), pack_f16(v.z * inv, v.w * inv)};
                    } else {
                        *reinterpret_cast<float4*>((g.dest == kSlot ? p.part : p.rowbuf) + e) = v;
                    }
                }
                if (!softmax_sync(mi, xphase)) return;
            }
        }
        wide_before = wide;
        tcgen05_fence_before();
        warp_arrive(&mi->segempty[slot]);
    }
}

// ---- matrix instructions -------------------------------------------------------

template <int FMT>
__device__ void mma_role(const Params& p, Misc* mi, unsigned char* smem) {
    constexpr int ring = Layout<FMT>::ring;
    constexpr uint32_t id_qk = mma_idesc_f16(128, 128, false), id_pv = mma_idesc_f16(128, 128, true);
    const int lane = threadIdx.x & 31;
    const uint32_t q_addr = smem_addr(smem), k_addr = q_addr + Layout<FMT>::tiles,
                   v_addr = q_addr + Layout<FMT>::v_tiles;
    uint32_t n_k = 0, n_v = 0, ph[2][2] = {};  // tiles of K and V; weights taken per stream and half
    auto wait_tile = [&](int v, uint32_t e) {
        return warp_wait(&mi->full[v][e % ring], (e / ring) & 1, mi);
    };
    // descriptors differ by constants: one addition each, in uniform registers
    const uint32_t leader = elect_one();
    const uint64_t q_desc = smem_desc(q_addr, 16, 1024), k_desc = smem_desc(k_addr, 16, 1024),
                   v_desc = smem_desc(v_addr, kHalfTile, 1024);
    // scores [row][position] = q K^T; thin units: [position][row] = K q^T
    auto scores = [&](int stream, int qslot, uint32_t e, bool thin, uint32_t idesc) {
        tcgen05_fence_after();
        const uint64_t q = q_desc + qslot * (kTileBytes >> 4), k = k_desc + (e % ring) * (kTileBytes >> 4);
        const uint64_t a = thin ? k : q, b = thin ? q : k;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t off = ((i >> 2) * kHalfTile + (i & 3) * 32) >> 4;
            mma_f16_ss(kTmem + stream * 128, a + off, b + off, idesc, i > 0, leader);
        }
        mma_commit(&mi->sfull[stream], leader);
    };
    // the next weights of this stream times V, half a tile's at a time
    auto pv = [&](int stream, uint32_t e, bool first) {
        const uint64_t b = v_desc + (e % ring) * (kTileBytes >> 4);
        const uint32_t o = kTmem + 256 + stream * 128, w = kTmem + stream * 128;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
            if (!warp_wait(&mi->pready[stream][h], ph[stream][h]++ & 1, mi)) return false;
            tcgen05_fence_after();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                mma_f16_ts(o, w + (4 * h + i) * 8, b + (4 * h + i) * (2048 >> 4), id_pv, !first || h > 0 || i > 0, leader);
            mma_commit(&mi->odone[stream][h], leader);
        }
        return true;
    };
    // thin units: sums [channel][row] += V^T w^T
    const uint64_t w_desc = smem_desc(q_addr + kTileBytes, 16, 1024);
    auto pv_thin = [&](int stream, uint32_t e, bool first, uint32_t idesc) {
        const uint64_t a = v_desc + (e % ring) * (kTileBytes >> 4), b = w_desc + stream * (kThinRows * 256 >> 4);
        if (!warp_wait(&mi->pready[stream][1], ph[stream][1]++ & 1, mi)) return false;
        tcgen05_fence_after();
#pragma unroll
        for (int i = 0; i < 8; ++i)
            mma_f16_ss(kTmem + 256 + stream * 128, a + i * (2048 >> 4),
                       b + (((i >> 2) * (kThinRows * 128) + (i & 3) * 32) >> 4),
                       idesc, !first || i > 0, leader);
        mma_commit(&mi->odone[stream][1], leader);
        return true;
    };
    auto release = [&](int v, uint32_t e) { mma_commit(&mi->empty[v][e % ring], leader); };
    // fp16 V rows that no row of the unit sees may hold anything (the end of a
    // page, tokens that left the window): 0 * NaN would reach the sums
    auto clean = [&](int4 seen, int tile, uint32_t e) {
        if (FMT != kF16) return;  // the conversion writes zeros there
        const int j0 = tile * kTile;
        const int lo = seen.x - j0, hi = seen.y - j0, fk = seen.z - j0, pfx = seen.w - j0;
        if ((lo <= 0 && hi >= kTile - 1) || (fk <= 0 && pfx >= kTile)) return;
        unsigned char* v = smem + Layout<FMT>::v_tiles + (e % ring) * kTileBytes + (lane & 7) * 16;
#pragma unroll 4
        for (int r = lane >> 3; r < kTile; r += 4) {
            if (!((r >= lo && r <= hi) || (r >= fk && r < pfx))) {
                *reinterpret_cast<uint4*>(v + r * 128) = uint4{0, 0, 0, 0};
                *reinterpret_cast<uint4*>(v + kHalfTile + r * 128) = uint4{0, 0, 0, 0};
            }
        }
        fence_async_smem();
        __syncwarp();
    };
    for (uint32_t k = 0, qk_seg = 0;; ++k) {
        const int slot = k % kSegs;
        if (!warp_wait(&mi->segfull[slot], (k / kSegs) & 1, mi)) return;
        const Segment& g = mi->seg[slot];
        if (!g.valid) return;
        // loads that the compiler then knows to be uniform
        const int t0 = __shfl_sync(kFull, g.t0, 0), n = __shfl_sync(kFull, g.t1, 0) - t0;
        const TileList tile(g);
        const int4 seen = {g.vlo, g.vhi, g.fk, g.pfx};
        if (n > 0) {
            if (!warp_wait(&mi->qfull, qk_seg++ & 1, mi)) return;
            // K of tile i + L and V of tile i, in the order they are copied
            const int mode = __shfl_sync(kFull, g.mode, 0), L = mode == kWide ? 1 : 2;
            const bool thin = mode == kThin;
            const uint32_t id_s = thin ? mma_idesc_f16(128, kThinRows, false) : id_qk;
#pragma unroll 1
            for (int i = -L; i < n; ++i) {
                const bool more = i + L < n;
                if (i >= 0) {
                    if (!wait_tile(1, n_v)) return;
                    clean(seen, tile(t0 + i), n_v);
                }
#pragma unroll 1
                for (int turn = 0; turn < 3 - L; ++turn) {
                    const int s = mode == kWide ? turn : i & 1;
                    if (i >= 0 && !(thin ? pv_thin(s, n_v, i < L, mma_idesc_f16(128, kThinRows, false) | (1u << 15))
                                         : pv(s, n_v, i < L)))
                        return;
                    if (more) {
                        if (turn == 0 && !wait_tile(0, n_k)) return;
                        scores(s, turn, n_k, thin, id_s);
                    }
                }
                if (i >= 0) release(1, n_v++);
                if (more) release(0, n_k++);
                if (i + L + 1 == n) mma_commit(&mi->qempty, leader);
            }
        }
        warp_arrive(&mi->segempty[slot]);
    }
}

// ---- copies --------------------------------------------------------------------

// Order of the copies: K of the first L tiles (wide units 1, others 2),
// then V_i, K_{i + L} for every tile i. K and V have rings of their own, so
// that each barrier's phases have one waiter that sees every one of them:
// a parity says nothing to a waiter that may be two phases behind.
//
// One warp copies K (and the queries), one V: a copy takes its warp some 120
// clocks to issue, and pages of 16 positions mean 16 copies for a tile of each.
template <int FMT>
__device__ void copy_role(const Params& p, Misc* mi, unsigned char* smem, const Maps& maps, bool is_v) {
    constexpr int ring = FMT == kF16 ? Layout<FMT>::ring : kRaw;
    const int lane = threadIdx.x & 31;
    const int sub_shift = 7 - p.box_shift, subs = 1 << sub_shift;    // boxes of a tile: 1 to 8
    const int sub = FMT == kF16 ? lane >> 1 & 7 : lane & 7;          // this lane's box
    const int part = FMT == kF16 ? lane & 1 : lane >> 3 & 1;         // half of the channels; codes or scales
    const bool mine = sub < subs && lane < 16;
    uint32_t pos = 0, q_seg = 0;  // tiles and query loads issued so far
    uint32_t thin = 0;            // 1 + the last thin segment
    uint64_t* const fulls = FMT == kF16 ? mi->full[is_v] : mi->rfull[is_v];
    uint64_t* const empties = FMT == kF16 ? mi->empty[is_v] : mi->rempty[is_v];
#pragma unroll 1
    for (uint32_t k = 0;; ++k) {
        const int slot = k % kSegs;
        if (!warp_wait(&mi->segfull[slot], (k / kSegs) & 1, mi)) break;
        const Segment& g = mi->seg[slot];
        if (!g.valid) break;
        const int t0 = g.t0, n = g.t1 - t0, mode = g.mode;
        bool ok = true;
        if (n > 0) {
            const TileList tile(g);
            const int vlo = g.vlo, vhi = g.vhi, fk = g.fk, pfx = g.pfx, head = g.head, tok0 = g.tok0;
            const KeySet& ks = p.set[g.set];
            const int* const table = ks.tables + static_cast<size_t>(g.seq) * ks.width;
            // Pages of 32 boxes (of 32 / subs tiles), one per lane: the page
            // number, -1 if it is none, -2 where nothing is seen.
            auto look = [&](int batch) {
                const int q = batch * 32 + lane, i = q >> sub_shift;
                if (i >= n) return -2;
                const int j = tile(t0 + i) * kTile + ((q & (subs - 1)) << p.box_shift), e = j + p.box_rows - 1;
                if (!((e >= vlo && j <= vhi) || (e >= fk && j < pfx))) return -2;
                return max(__ldg(table + p.by_block(j)), -1);
            };
            // its row in the caches; the row past the last reads as zeros
            auto place = [&](int page, int batch) {
                if (page == -2) return p.total_rows;
                if (page < 0 || page >= p.num_blocks) {
                    atomicCAS(&g_attention_error, 0, static_cast<int>(kDevBadBlock));
                    return p.total_rows;
                }
                const int q = batch * 32 + lane;
                const int j = tile(t0 + (q >> sub_shift)) * kTile + ((q & (subs - 1)) << p.box_shift);
                return (page * p.n_kv + head) * p.block_size + j - p.by_block(j) * p.block_size;
            };
            int batch = -1, ahead = look(0), rows = 0;
            if (!is_v) {
                // queries: the last segment's score tiles are done with them
                if (q_seg > 0 && !warp_wait(&mi->qempty, (q_seg - 1) & 1, mi)) break;
                if (mode == kWide && thin && k - (thin - 1) < kSegs &&
                    !warp_wait(&mi->segempty[(thin - 1) % kSegs], ((thin - 1) / kSegs) & 1, mi))
                    break;  // a thin segment still uses the second tile's place
                const int copies = mode == kWide ? 2 : 1, toks = mode == kThin ? p.thin_per : p.per;
                if (lane == 0) mbar_arrive_expect_tx(&mi->qfull, static_cast<uint32_t>(copies * toks * p.group * 256));
                __syncwarp();
                if (lane < 2 * copies) {
                    const int c = lane >> 1, half = lane & 1;
                    tma_load_3d(smem + c * kTileBytes + half * kHalfTile, &maps.q[mode == kThin], half * 64,
                                head * p.group, tok0 + c * toks, &mi->qfull);
                }
                ++q_seg;
            }
            const int L = mode == kWide ? 1 : 2;
#pragma unroll 1
            for (int i = -L; i < n; ++i) {
                const int it = is_v ? i : i + L;  // this warp's tile now
                if (it < 0 || it >= n) continue;
                const uint32_t e = pos;
                if (it << sub_shift >> 5 != batch) {
                    ++batch;
                    rows = place(ahead, batch);
                    ahead = look(batch + 1);
                }
                const uint32_t st = e % ring;
                if (e >= ring && !warp_wait(&empties[st], (e / ring - 1) & 1, mi)) {
                    ok = false;
                    break;
                }
                const int row = __shfl_sync(kFull, rows, ((it << sub_shift) + sub) & 31);
                uint64_t* const full = &fulls[st];
                const CUtensorMap* map = is_v ? &maps.v : &maps.k;
                if (FMT == kF16) {
                    if (lane == 0) mbar_arrive_expect_tx(full, kTileBytes);
                    __syncwarp();
                    if (mine)
                        tma_load_2d(smem + (is_v ? Layout<FMT>::v_tiles : Layout<FMT>::tiles) + st * kTileBytes +
                                        part * kHalfTile + (sub << p.box_shift) * 128,
                                    map, part * 64, row, full);
                } else {
                    const bool there = mine && row != p.total_rows;
                    const unsigned here = __ballot_sync(kFull, there && part == 0);
                    if (lane == 0) {
                        mi->bad[is_v][st] = ~here & ((1u << subs) - 1);
                        mbar_arrive_expect_tx(full, kRawBytes + (__popc(here) << p.box_shift) * 2);
                    }
                    __syncwarp();
                    if (mine && part == 0)
                        tma_load_2d(smem + Layout<FMT>::raw + (is_v * kRaw + st) * kRawBytes + (sub << p.box_shift) * kHeadDim, map, 0, row,
                                    full);
                    if (there && part == 1)
                        bulk_g2s_plain(smem + Layout<FMT>::raw_scale + (is_v * kRaw + st) * 256 + (sub << p.box_shift) * 2,
                                       (is_v ? p.v_scale : p.k_scale) + row, p.box_rows * 2, full);
                }
                __syncwarp();
                ++pos;
            }
        }
        if (!ok) break;
        if (mode == kThin) thin = k + 1;
        warp_arrive(&mi->segempty[slot]);
    }
    // Leave no copy in flight: if a wait runs out, here or in another warp and
    // later, nobody else waits for them. A slot's earlier copy was done before its
    // latest one was issued, and none is issued afterwards, so each parity names it.
#pragma unroll 1
    for (uint32_t e = pos > ring ? pos - ring : 0; e < pos; ++e)
#pragma unroll 1
        for (uint32_t i = 0; i < kPolls && !mbar_try_wait(&fulls[e % ring], (e / ring) & 1); ++i) {}
    if (q_seg > 0)
#pragma unroll 1
        for (uint32_t i = 0; i < kPolls && !mbar_try_wait(&mi->qfull, (q_seg - 1) & 1); ++i) {}
}

// ---- INT8 conversion -------------------------------------------------------------

// Codes to fp16 integers (exact) in the swizzled tile, scales to fp32; one
// warpgroup for K, one for V (a single one took 4200 clocks for a tile of both,
// three times what its bytes take from memory). V's
// scales go out before V's codes wait for room, since the softmax of the tile
// needs them; they are divided by the power of two above the segment's largest
// so far, so that weight * scale fits fp16. Rows that no row of the unit sees,
// and rows of pages that are not there, become zeros with scale zero.
__device__ void convert_role(const Params& p, Misc* mi, unsigned char* smem, bool is_v) {
    constexpr uint32_t ring = Layout<kI8>::ring;
    Scales* const scales = reinterpret_cast<Scales*>(smem + Layout<kI8>::scales);
    const int t = threadIdx.x & 127;
    // 16 channels (chunk c) of eight rows. A quarter warp holds chunks of one
    // half of rows q and q ^ 5: both the swizzled codes it reads and the
    // swizzled tile it writes then spread over all banks.
    const int lane = t & 31;
    const int c = (lane & 3) + (lane >> 1 & 4), turn = lane & 4 ? 5 : 0, x = (c & 3) * 2;
    const int r0 = (t >> 5) * 32 + (lane >> 4);
    auto row_of = [&](int i) { return (r0 + (i >> 1) * 8 + (i & 1) * 2) ^ turn; };
    uint32_t done = 0;  // tiles
    int top = 0;        // V's exponent
#pragma unroll 1
    for (uint32_t k = 0;; ++k) {
        const int slot = k % kSegs;
        if (!warp_wait(&mi->segfull[slot], (k / kSegs) & 1, mi)) return;
        const Segment& g = mi->seg[slot];
        if (!g.valid) return;
        const int t0 = g.t0, n = g.t1 - t0;
        const TileList tile(g);
        const int4 range = {g.vlo, g.vhi, g.fk, g.pfx};
        top = -60;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const uint32_t m = done++;
            const int st = m % kRaw, j0 = tile(t0 + i) * kTile;
            if (!warp_wait(&mi->rfull[is_v][st], (m / kRaw) & 1, mi)) return;
            const unsigned char* src = smem + Layout<kI8>::raw + (is_v * kRaw + st) * kRawBytes;
            const __half* scale = reinterpret_cast<const __half*>(smem + Layout<kI8>::raw_scale + (is_v * kRaw + st) * 256);
            const uint32_t bad = mi->bad[is_v][st];
            const int lo = range.x - j0, hi = range.y - j0, fk = range.z - j0, pfx = range.w - j0;
            const bool all = __all_sync(kFull, ((lo <= 0 && hi >= kTile - 1) || (fk <= 0 && pfx >= kTile)) && bad == 0);
            auto seen = [&](int r) {
                return ((r >= lo && r <= hi) || (r >= fk && r < pfx)) && !((bad >> (r >> p.box_shift)) & 1);
            };
            const int at = m % kScales, d = m % ring;
            const bool mine_seen = all || seen(t);
            const float sc = mine_seen ? __half2float(scale[t]) : 0.f;
            if (!is_v) {
                scales->k[at][t] = sc * p.kf;
            } else {
                const int r4 = lane * 4;
                const uint2 raw = *reinterpret_cast<const uint2*>(scale + r4);
                const float2 a = __half22float2(__habs2(as_h2(raw.x))), b = __half22float2(__habs2(as_h2(raw.y)));
                float most = fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y));
                if (!all)
                    most = fmaxf(fmaxf(seen(r4) ? a.x : 0.f, seen(r4 + 1) ? a.y : 0.f),
                                 fmaxf(seen(r4 + 2) ? b.x : 0.f, seen(r4 + 3) ? b.y : 0.f));
                const uint32_t bits = __reduce_max_sync(kFull, __float_as_uint(most));
                top = max(top, min(static_cast<int>(bits >> 23) - 126, 17));  // 17: no finite scale
                scales->v[at][t] = sc * __int_as_float((127 - top) << 23);
                scales->v_exp[at] = top;
                warp_arrive(&mi->vscale[at]);
            }
            uint4 in[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int r = row_of(q);
                in[q] = *reinterpret_cast<const uint4*>(src + r * kHeadDim + ((c ^ (r & 7)) << 4));
            }
            warp_arrive(&mi->rempty[is_v][st]);
            if (m >= ring && !warp_wait(&mi->empty[is_v][d], (m / ring - 1) & 1, mi)) return;
            unsigned char* dst = smem + (is_v ? Layout<kI8>::v_tiles : Layout<kI8>::tiles) + d * kTileBytes + (c >> 2) * kHalfTile;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int r = row_of(q);
                half2 o[4];
                unsigned char* line = dst + r * 128;
                i8x4_to_h2(in[q].x, o[0], o[1]);
                i8x4_to_h2(in[q].y, o[2], o[3]);
                *reinterpret_cast<uint4*>(line + ((x ^ (r & 7)) << 4)) =
                    uint4{as_u32(o[0]), as_u32(o[1]), as_u32(o[2]), as_u32(o[3])};
                i8x4_to_h2(in[q].z, o[0], o[1]);
                i8x4_to_h2(in[q].w, o[2], o[3]);
                *reinterpret_cast<uint4*>(line + (((x + 1) ^ (r & 7)) << 4)) =
                    uint4{as_u32(o[0]), as_u32(o[1]), as_u32(o[2]), as_u32(o[3])};
            }
            if (!all) {
#pragma unroll 1
                for (int q = 0; q < 8; ++q) {
                    const int r = row_of(q);
                    if (seen(r)) continue;
                    *reinterpret_cast<uint4*>(dst + r * 128 + ((x ^ (r & 7)) << 4)) = uint4{0, 0, 0, 0};
                    *reinterpret_cast<uint4*>(dst + r * 128 + (((x + 1) ^ (r & 7)) << 4)) = uint4{0, 0, 0, 0};
                }
            }
            fence_async_smem();
            warp_arrive(&mi->full[is_v][d]);
        }
        warp_arrive(&mi->segempty[slot]);
    }
}

// ---- schedule --------------------------------------------------------------------

// Cost of a unit: its tiles (an empty one still writes its rows) behind what
// starting and finishing one takes. A tile weighs p.weight[mode], what it was
// measured to take; tile t of a unit lies at lead + t * weight and belongs to the
// CTA that this position belongs to.
__device__ __forceinline__ int unit_cost(const Params& p, const Segment& s) {
    return p.lead + max(s.nt, 1) * p.weight[s.mode];
}

// The units, laid end to end, are split over `ctas` CTAs, the first `more` of
// which take one more than the others. Each takes at least the heaviest tile's
// weight, so that from a split unit's first CTA to its last all have a tile of it.
// x / y; mostly both fit 32 bits, and 64-bit division is a long subroutine
__device__ __forceinline__ long long divide(long long x, long long y) {
    if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
    return x / y;
}
struct Split {
    long long each, more, ctas;
    __device__ Split(const Params& p, long long total, int heaviest)
        : ctas(max(min(static_cast<long long>(p.grid), divide(total, max(heaviest, 1))), 1LL)) {
        each = divide(total, ctas);
        more = total - each * ctas;
    }
    __device__ long long start(long long cta) const { return cta * each + min(cta, more); }
    __device__ int owner(long long x) const {
        const long long edge = more * (each + 1);
        return static_cast<int>(x < edge ? divide(x, each + 1) : more + divide(x - edge, each));
    }
};

// This CTA's share [start, start + count) of all units' tiles, and the unit it
// begins in: a block-wide prefix sum over the unit numbers.
template <int THREADS>
__device__ void plan(const Params& p, Misc* mi) {
    const int n_ids = p.set[0].n_ids + (p.n_sets > 1 ? p.set[1].n_ids : 0);
    const int chunk = (n_ids + THREADS - 1) / THREADS;
    const int id0 = threadIdx.x * chunk, id1 = min(id0 + chunk, n_ids);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long sum = 0, a = 0, at = 0;
    int heaviest = 0;
    Segment s;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {  // add up; then, in the thread that has it, find the CTA's first unit
#pragma unroll 1
        for (int id = id0; id < id1; ++id) {
            // with one number per thread the first pass has left it in s
            if ((pass == 0 || chunk > 1) && !make_unit(p, id, s)) continue;
            const int c = unit_cost(p, s);
            if (pass == 0) {
                sum += c;
                heaviest = max(heaviest, p.weight[s.mode]);
            } else if (a - at < static_cast<long long>(c) * p.n_kv) {
                const long long rest = a - at;
                mi->start_id = id;
                mi->start_head = static_cast<int>(divide(rest, c));
                mi->start_off = static_cast<int>(rest - static_cast<long long>(mi->start_head) * c);
                mi->first = s;
                break;
            } else {
                at += static_cast<long long>(c) * p.n_kv;
            }
        }
        if (pass == 1) break;
        long long incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(kFull, incl, d);
            if (lane >= d) incl += o;
        }
        heaviest = __reduce_max_sync(kFull, heaviest);
        if (lane == 31) {
            mi->scan[warp] = incl;
            mi->heavy[warp] = heaviest;
        }
        __syncthreads();
        long long total = 0;
#pragma unroll 1
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) at += mi->scan[w];
            total += mi->scan[w];
            heaviest = max(heaviest, mi->heavy[w]);
        }
        total *= p.n_kv;
        const Split split(p, total, heaviest);
        a = split.start(blockIdx.x);
        const long long e = blockIdx.x < split.ctas ? split.start(blockIdx.x + 1) : a;
        if (threadIdx.x == 0) {
            mi->start = a;
            mi->count = e - a;
            mi->total = total;
            mi->heaviest = heaviest;
        }
        at = (at + incl - sum) * p.n_kv;
        if (!(e > a && at <= a && a < at + sum * p.n_kv)) break;
    }
}

__device__ void schedule_role(const Params& p, Misc* mi) {
    const int lane = threadIdx.x & 31;
    long long left = mi->count, at = mi->start;
    const Split parts(p, mi->total, mi->heaviest);
    const int n_ids = p.set[0].n_ids + (p.n_sets > 1 ? p.set[1].n_ids : 0);
    int id = mi->start_id, head = mi->start_head, off = mi->start_off;
    bool split = false;
    Segment s = mi->first;
#pragma unroll 1
    for (uint32_t k = 0;;) {
        const int slot = k % kSegs;
        const int cost = unit_cost(p, s), weight = p.weight[s.mode], tiles = max(s.nt, 1);
        const int n = static_cast<int>(min(left, static_cast<long long>(cost - off)));
        // tiles that begin within [off, off + n)
        const int t0 = (max(off - p.lead, 0) + weight - 1) / weight;
        const int t1 = (max(off + n - p.lead, 0) + weight - 1) / weight;
        const bool last = left <= 0;
        if (last || t1 > t0) {
            const bool whole = t0 == 0 && t1 == tiles;
            // a whole segment may pass, seconds for one over millions of keys
            if (k >= kSegs && !warp_wait(&mi->segempty[slot], (k / kSegs - 1) & 1, mi, kPolls * 64)) break;
            if (lane == 0) {
                s.valid = !last;
                s.head = head;
                s.t0 = s.nt ? t0 : 0;
                s.t1 = s.nt ? t1 : 0;
                s.dest = !whole ? kSlot : p.shared ? kRowBuf : kDirect;
                mi->seg[slot] = s;
                if (!last && t0 == 0) {  // a split unit is finished by the owner of its last tile
                    const int to = whole ? -1 : parts.owner(at - off + cost - weight);
                    if (p.shared) p.units[static_cast<size_t>(id) * p.n_kv + head] = {static_cast<int>(blockIdx.x), to};
                    if (!whole) p.split[blockIdx.x] = {s.tok0, s.ntok, head, to};
                }
            }
            warp_arrive(&mi->segfull[slot]);
            if (last) break;
            split |= t0 == 0 && !whole;
            ++k;
        }
        at += n;
        left -= n;
        off = 0;
        if (left > 0 && ++head == p.n_kv) {
            head = 0;
            do ++id; while (id < n_ids && !make_unit(p, id, s));
            if (id >= n_ids) left = 0;
        }
    }
    if (!split && lane == 0) p.split[blockIdx.x] = {0, 0, 0, -1};
}

template <int FMT, bool MOD>
__global__ void __launch_bounds__(Layout<FMT>::threads, 1)
    attention_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
    using Lay = Layout<FMT>;
    extern __shared__ __align__(1024) unsigned char smem[];
    Misc* mi = reinterpret_cast<Misc*>(smem + Lay::misc);
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        const int readers = FMT == kF16 ? 11 : 19;  // warps that read a segment
        auto late = [&](Stall what) { return p.stall == what ? 1 : 0; };
        for (int v = 0; v < 2; ++v) {
            for (int i = 0; i < kMaxRing; ++i) {
                mbar_init(&mi->full[v][i], (FMT == kF16 ? 1 : 4) + late(v ? kStallV : kStallK));
                mbar_init(&mi->empty[v][i], 1);
            }
        }
        for (int i = 0; i < 2 * kRaw; ++i) {
            mbar_init(&mi->rfull[0][i], 1 + late(kStallRaw));
            mbar_init(&mi->rempty[0][i], 4);
        }
        mbar_init(&mi->qfull, 1 + late(kStallQuery));
        mbar_init(&mi->qempty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&mi->sfull[i], 1 + late(kStallScores));
            for (int h = 0; h < 2; ++h) {
                mbar_init(&mi->pready[i][h], 4 + late(kStallWeights));
                mbar_init(&mi->odone[i][h], 1 + late(kStallSums));
            }
        }
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(&mi->segfull[i], 1 + late(kStallSegment));
            mbar_init(&mi->segempty[i], readers);
        }
        for (int i = 0; i < kScales; ++i) mbar_init(&mi->vscale[i], 4);
        for (int i = 0; i < 2; ++i) mbar_init(&mi->tbar[i], 4);
        mbar_init(&mi->xbar, 8);
        mbar_init(&mi->drain, 1);
        mi->abort = 0;
        mi->first = Segment{};  // stays so in a CTA without a share
        mi->start_id = mi->start_head = mi->start_off = 0;
        fence_barrier_init();
        tma_prefetch_map(&maps.k);
        tma_prefetch_map(&maps.v);
    }
    if (warp == 9) tmem_alloc(&mi->tmem, 512);
    grid_dependency_wait();
    grid_launch_dependents();
    plan<Lay::threads>(p, mi);
    if (FMT != kF16 && threadIdx.x < kTile / 2) reinterpret_cast<Scales*>(smem + Lay::scales)->ones[threadIdx.x] = 1.f;
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    // All columns were asked for, so they start at 0: a constant, which keeps
    // the matrix instructions' operands in uniform registers. (Checked: any
    // other answer ends the block as an expired wait does.)
    if (mi->tmem != kTmem) *reinterpret_cast<volatile int*>(&mi->abort) = 1;

    if (warp < 8) {
        regs_inc<Lay::softmax_regs>();
        softmax_role<FMT, MOD>(p, mi, smem);
    } else if (warp < 12) {
        regs_dec<Lay::other_regs>();
        if (warp == 8) {
            copy_role<FMT>(p, mi, smem, maps, false);
        } else if (warp == 11) {
            copy_role<FMT>(p, mi, smem, maps, true);
        } else if (warp == 9) {
            mma_role<FMT>(p, mi, smem);
            __syncwarp();
            mma_commit(&mi->drain, elect_one());  // leave no product running, as for the copies
#pragma unroll 1
            for (uint32_t i = 0; i < kPolls && !mbar_try_wait(&mi->drain, 0); ++i) {}
        } else if (warp == 10) {
            schedule_role(p, mi);
        }
    } else {
        if constexpr (FMT != kF16) {
            regs_dec<Lay::convert_regs>();
            convert_role(p, mi, smem, warp >= 16);
        }
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 9) {
        tcgen05_fence_after();
        tmem_dealloc(mi->tmem, 512);
        if (mi->abort) atomicCAS(&g_attention_error, 0, static_cast<int>(kDevWaitTimeout));
    }
}

// ---- joining -----------------------------------------------------------------------

// Adds the partial states of one row, this lane's four channels, in CTA order.
struct Join {
    float m = -INFINITY, l = 0.f;
    float4 v = {0.f, 0.f, 0.f, 0.f};
    __device__ void add(const float2* ml, const float* part, size_t r, int lane) {
        const float2 e = ml[r];
        if (e.y == 0.f) return;
        const float4 o = *reinterpret_cast<const float4*>(part + r * kHeadDim + lane * 4);
        const float up = fmaxf(m, e.x);
        const float a = m == -INFINITY ? 0.f : fast_exp2(m - up), b = fast_exp2(e.x - up);
        m = up;
        l = l * a + e.y * b;
        v = {v.x * a + o.x * b, v.y * a + o.y * b, v.z * a + o.z * b, v.w * a + o.w * b};
    }
    // The partial states of a unit's row in the CTAs first .. last. A lane reads
    // one CTA's state, then the sums come four at a time: one after the other, each
    // behind its state, a unit that 18 CTAs share took 53 us in place of 32.
    // A CTA that gave up (a wait ran out) may have left its entries unwritten:
    // what is out of range is left out, and the error word has told.
    __device__ void add_slots(const Params& p, int first, int last, int unit_row, int lane) {
        if (first < 0 || last >= p.grid || unit_row >= p.slot_rows) return;
        auto slot = [&](int c) { return static_cast<size_t>(2 * c + (c == first)) * p.slot_rows + unit_row; };
        for (int c0 = first; c0 <= last; c0 += 32) {
            const int n = min(32, last - c0 + 1);
            const float2 e = lane < n ? p.part_ml[slot(c0 + lane)] : float2{-INFINITY, 0.f};
            float up = e.y == 0.f ? -INFINITY : e.x, sum;
#pragma unroll
            for (int d = 16; d; d >>= 1) up = fmaxf(up, __shfl_xor_sync(kFull, up, d));
            up = fmaxf(up, m);
            const float a = m == -INFINITY ? 0.f : fast_exp2(m - up), f = e.y == 0.f ? 0.f : fast_exp2(e.x - up);
            sum = e.y * f;
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
            m = up;
            l = l * a + sum;
            v = {v.x * a, v.y * a, v.z * a, v.w * a};
            for (int i = 0; i < n; i += 4) {
                float4 o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o[k] = *reinterpret_cast<const float4*>(p.part + slot(c0 + min(i + k, n - 1)) * kHeadDim + lane * 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float b = __shfl_sync(kFull, f, (i + k) & 31);
                    if (i + k < n && b != 0.f)
                        v = {v.x + o[k].x * b, v.y + o[k].y * b, v.z + o[k].z * b, v.w + o[k].w * b};
                }
            }
        }
    }
    __device__ void store(const Params& p, size_t row, int lane) {
        const float inv = over_sum(l);
        uint2 u;
        u.x = pack_f16(v.x * inv, v.y * inv);
        u.y = pack_f16(v.z * inv, v.w * inv);
        *reinterpret_cast<uint2*>(p.out + row * kHeadDim + lane * 4) = u;
    }
};

// One warp per row of a split unit; blockIdx.x is the CTA the unit starts in.
__global__ void __launch_bounds__(256) join_split_kernel(const __grid_constant__ Params p) {
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 u = p.split[blockIdx.x];
    // (entries that a CTA which gave up never wrote hold anything)
    if (u.w >= 0 && u.x >= 0 && u.y >= 0 && u.y <= 2 * (kTile / p.group) && u.x <= p.n_tokens - u.y && u.z >= 0 &&
        u.z < p.n_kv) {
        const int rows = u.y * p.group;
        for (int r = blockIdx.y * 8 + warp; r < rows; r += gridDim.y * 8) {
            Join j;
            j.add_slots(p, blockIdx.x, u.w, r, lane);
            const int tk = r / p.group;
            j.store(p, static_cast<size_t>(u.x + tk) * p.n_heads + u.z * p.group + r - tk * p.group, lane);
        }
    }
    if (p.zero_tail) {  // tokens of no sequence
        const KeySet& k = p.set[0];
        const long long lo = cu_at(k, 0, p.n_tokens), hi = cu_at(k, k.n_seq, p.n_tokens);
        const long long pad = (lo + p.n_tokens - hi) * p.n_heads;
        const long long step = static_cast<long long>(gridDim.x) * gridDim.y * 8;
        for (long long i = (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * 8 + warp; i < pad; i += step) {
            const long long row = i < lo * p.n_heads ? i : i + (hi - lo) * p.n_heads;
            *reinterpret_cast<uint2*>(p.out + row * kHeadDim + lane * 4) = uint2{0, 0};
        }
    }
}

// One warp per (token, query head): the shared prefix's state, then its own.
__global__ void __launch_bounds__(256) join_rows_kernel(const __grid_constant__ Params p) {
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (row >= static_cast<long long>(p.n_tokens) * p.n_heads) return;
    const int tok = static_cast<int>(row / p.n_heads), hq = static_cast<int>(row - static_cast<long long>(tok) * p.n_heads);
    const int h = hq / p.group, g = hq - h * p.group;
    const int unit = 2 * (kTile / p.group);
    Join j;
    const KeySet& k = p.set[0];
    int lo = 0, hi = k.n_seq - 1;  // the group that holds this token
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu_at(k, mid, p.n_tokens) <= tok) lo = mid; else hi = mid - 1;
    }
    const int c0 = cu_at(k, lo, p.n_tokens);
    if (k.n_seq > 0 && tok >= c0 && tok < cu_at(k, lo + 1, p.n_tokens)) {
        const int at = (tok - c0) / unit;
        const int id = at == 0 ? lo : k.n_seq + c0 / unit + at - 1;
        const int2 u = p.units[static_cast<size_t>(id) * p.n_kv + h];
        if (u.y < 0)
            j.add(p.row_ml, p.rowbuf, row, lane);
        else
            j.add_slots(p, u.x, u.y, (tok - c0 - at * unit) * p.group + g, lane);
    }
    const int2 u = p.units[static_cast<size_t>(k.n_ids + tok) * p.n_kv + h];
    if (u.y < 0)
        j.add(p.row_ml, p.rowbuf, static_cast<size_t>(p.n_tokens) * p.n_heads + row, lane);
    else
        j.add_slots(p, u.x, u.y, g, lane);
    j.store(p, row, lane);
}

// ---- host ----------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, looked up in the driver once (the library does not
// link against it, so it loads on machines without a GPU).
EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

bool encode(CUtensorMap* m, CUtensorMapDataType dt, int rank, const void* base, const cuuint64_t* dims,
            const cuuint64_t* strides, const cuuint32_t* box, bool swizzle, std::string& err) {
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = encode_fn()(m, dt, rank, const_cast<void*>(base), dims, strides, box, one,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) err = "cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")";
    return r == CUDA_SUCCESS;
}

struct Plan {  // sizes that the workspace and the launch agree on
    int per, unit, n_ids0, n_ids1, slot_rows;
    size_t part, ml, split, rowbuf, row_ml, units, bytes;
};
Plan make_plan(int64_t n_tokens, int64_t n_heads, int64_t n_kv, int64_t n_seq0, bool shared, int grid) {
    Plan w{};
    const int64_t group = n_heads / n_kv;
    w.per = static_cast<int>(kTile / group);
    w.unit = 2 * w.per;
    w.n_ids0 = static_cast<int>(n_tokens / w.unit + n_seq0);
    w.n_ids1 = shared ? static_cast<int>(n_tokens) : 0;
    w.slot_rows = static_cast<int>(std::min<int64_t>(w.unit, n_tokens) * group);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at = align_up(at + bytes, 256);
        return o;
    };
    w.part = take(size_t{2} * grid * w.slot_rows * kHeadDim * 4);
    w.ml = take(size_t{2} * grid * w.slot_rows * sizeof(float2));
    w.split = take(size_t{1} * grid * sizeof(int4));
    if (shared) {
        const size_t rows = static_cast<size_t>(n_tokens) * n_heads;
        w.rowbuf = take(2 * rows * kHeadDim * 4);
        w.row_ml = take(2 * rows * sizeof(float2));
        w.units = take(static_cast<size_t>(w.n_ids0 + w.n_ids1) * n_kv * sizeof(int2));
    }
    w.bytes = at;
    return w;
}

template <int FMT, bool MOD>
lik_status launch(const Maps& maps, const Params& p, cudaStream_t stream, std::string& err) {
    using Lay = Layout<FMT>;
    auto kern = attention_kernel<FMT, MOD>;
    static std::mutex mu;
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev & 63]) {
            cudaFuncAttributes fa;
            e = cudaFuncGetAttributes(&fa, kern);
            if (e == cudaSuccess && fa.numRegs != Lay::base) {
                err = "attention kernel: built with " + std::to_string(fa.numRegs) + " registers, its shares need " +
                      std::to_string(Lay::base);
                return LIK_ERR_CUDA;
            }
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay::bytes);
            if (e == cudaSuccess) ready[dev & 63] = true;
        }
    }
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(p.grid);
        cfg.blockDim = dim3(Lay::threads);
        cfg.dynamicSmemBytes = Lay::bytes;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, kern, maps, p);
        if (e == cudaSuccess) {
            cfg.blockDim = dim3(256);
            cfg.dynamicSmemBytes = 0;
            if (p.shared) {
                const long long rows = static_cast<long long>(p.n_tokens) * p.n_heads;
                cfg.gridDim = dim3(static_cast<unsigned>((rows + 7) / 8));
                e = cudaLaunchKernelEx(&cfg, join_rows_kernel, p);
            } else {
                // two rows per warp: four took 32 us in place of 27 for 42 tokens over 1798 keys,
                // one 161 us in place of 153 for a prompt of 4096 after a pause (idle blocks)
                cfg.gridDim = dim3(p.grid, static_cast<unsigned>((p.slot_rows + 15) / 16));
                e = cudaLaunchKernelEx(&cfg, join_split_kernel, p);
            }
        }
    }
    if (e != cudaSuccess) {
        err = std::string("attention launch: ") + cudaGetErrorString(e);
        return LIK_ERR_CUDA;
    }
    return LIK_OK;
}

thread_local int next_stall = kNoStall;

}  // namespace

void stall_next_attention(int what) { next_stall = what; }

size_t attention_workspace_bytes(int64_t n_tokens, int64_t n_heads, int64_t n_kv, int64_t n_groups, bool shared,
                                 int sm_count) {
    return make_plan(n_tokens, n_heads, n_kv, shared ? n_groups : 0, shared, sm_count).bytes;
}

void* attention_error_word(std::string& err) {
    void* a = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&a, g_attention_error);
    if (e != cudaSuccess) err = std::string("cudaGetSymbolAddress: ") + cudaGetErrorString(e);
    return e == cudaSuccess ? a : nullptr;
}

lik_status launch_attention(const AttentionArgs& a, cudaStream_t stream, std::string& err) {
    DeviceInfo di;
    if (!device_info(di, err)) return LIK_ERR_CUDA;
    if (!encode_fn()) {
        err = "cuTensorMapEncodeTiled not found in the driver";
        return LIK_ERR_CUDA;
    }
    const bool shared = a.prefix_tables != nullptr;
    const Plan w = make_plan(a.n_tokens, a.n_heads, a.n_kv_heads, shared ? a.n_groups : a.n_seqs, shared, di.sm_count);
    if (!a.workspace || a.workspace_bytes < w.bytes) {
        err = "attention workspace of " + std::to_string(w.bytes) + " bytes needed";
        return LIK_ERR_WORKSPACE;
    }
    Params p{};
    if (shared) {
        p.set[0] = {a.cu_seqlens, a.prefix_lens, a.prefix_tables, a.context_lens, static_cast<int>(a.n_groups),
                    static_cast<int>(a.prefix_blocks), w.n_ids0, 0};
        p.set[1] = {nullptr, a.context_lens, a.block_tables, nullptr, static_cast<int>(a.n_tokens),
                    static_cast<int>(a.max_blocks), w.n_ids1, 0};
        p.n_sets = 2;
        p.extra_most = static_cast<int>(a.max_blocks * a.block_size);
    } else {
        p.set[0] = {a.cu_seqlens, a.context_lens, a.block_tables, nullptr, static_cast<int>(a.n_seqs),
                    static_cast<int>(a.max_blocks), w.n_ids0, a.causal ? 1 : 0};
        p.n_sets = 1;
        p.prefix_lens = a.prefix_lens;
        p.first_keys = a.first_keys;
        p.window = static_cast<int>(a.window);
    }
    p.slopes = a.alibi_slopes;
    p.kf = a.softcap > 0.f ? a.softmax_scale / a.softcap : a.softmax_scale * kLog2e;
    p.cap = a.softcap;
    p.n_tokens = static_cast<int>(a.n_tokens);
    p.n_heads = static_cast<int>(a.n_heads);
    p.n_kv = static_cast<int>(a.n_kv_heads);
    p.group = p.n_heads / p.n_kv;
    p.per = w.per;
    p.thin_per = kThinRows / p.group;
    // clocks measured per tile, in units of 270: wide 4300 (fp16) and 6500 (INT8,
    // converted on the way), paired 2500 and 3800, thin 2700 (what its bytes take
    // from memory) and 3800; 7500 to start and finish a unit
    const bool int8 = a.fmt != kF16;
    p.lead = 28;
    p.weight[kWide] = int8 ? 24 : 16;
    p.weight[kPaired] = int8 ? 14 : 9;
    p.weight[kThin] = int8 ? 14 : 10;
    p.by_group = make_div(p.group);
    p.by_unit = make_div(w.unit);
    p.by_block = make_div(static_cast<uint32_t>(a.block_size));
    p.num_blocks = static_cast<int>(a.num_blocks);
    p.block_size = static_cast<int>(a.block_size);
    p.box_rows = std::min(kTile, p.block_size & -p.block_size);  // boxes never cross a page
    for (p.box_shift = 0; 1 << p.box_shift < p.box_rows; ++p.box_shift) {}
    p.total_rows = static_cast<int>(a.num_blocks * a.n_kv_heads * a.block_size);
    p.k_scale = static_cast<const __half*>(a.k_scale);
    p.v_scale = static_cast<const __half*>(a.v_scale);
    p.out = static_cast<__half*>(a.out);
    p.shared = shared;
    p.zero_tail = a.zero_tail;
    p.slot_rows = w.slot_rows;
    p.grid = di.sm_count;
    p.stall = next_stall;
    next_stall = kNoStall;
    unsigned char* ws = static_cast<unsigned char*>(a.workspace);
    p.part = reinterpret_cast<float*>(ws + w.part);
    p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
    p.split = reinterpret_cast<int4*>(ws + w.split);
    p.rowbuf = reinterpret_cast<float*>(ws + w.rowbuf);
    p.row_ml = reinterpret_cast<float2*>(ws + w.row_ml);
    p.units = reinterpret_cast<int2*>(ws + w.units);

    Maps maps;
    for (int i = 0; i < 2; ++i) {
        const int toks = i ? p.thin_per : p.per;
        if (toks == 0) {
            maps.q[i] = maps.q[0];
            continue;
        }
        const cuuint64_t dims[3] = {kHeadDim, static_cast<cuuint64_t>(a.n_heads), static_cast<cuuint64_t>(a.n_tokens)};
        const cuuint64_t strides[2] = {kHeadDim * 2, static_cast<cuuint64_t>(a.n_tokens > 1 ? a.q_token_stride : a.n_heads * kHeadDim) * 2};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(toks)};
        if (!encode(&maps.q[i], CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.q, dims, strides, box, true, err)) return LIK_ERR_CUDA;
    }
    const bool f16 = a.fmt == kF16;
    const cuuint64_t dims[2] = {kHeadDim, static_cast<cuuint64_t>(p.total_rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(kHeadDim) * (f16 ? 2 : 1)};
    const cuuint32_t box[2] = {f16 ? 64u : 128u, static_cast<cuuint32_t>(p.box_rows)};
    const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    if (!encode(&maps.k, dt, 2, a.k, dims, strides, box, true, err) || !encode(&maps.v, dt, 2, a.v, dims, strides, box, true, err))
        return LIK_ERR_CUDA;
    const bool mod = p.cap > 0.f || p.slopes;
    if (f16) return mod ? launch<kF16, true>(maps, p, stream, err) : launch<kF16, false>(maps, p, stream, err);
    return mod ? launch<kI8, true>(maps, p, stream, err) : launch<kI8, false>(maps, p, stream, err);
}

}  // namespace lik
