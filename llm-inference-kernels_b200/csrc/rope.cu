// Append to a paged cache with the position rotation on the way.
//
//   angle = position[axis(f)] * inv_freq[f]
//   (a, b) -> (a cos - b sin, b cos + a sin)
//
// over the channel pairs f of the first 2 r channels (r = number of
// frequencies): (f, f + r), or (2f, 2f + 1) when interleaved; the other
// channels pass. Frequencies belong to position axes in consecutive sections
// (one axis: text; three: time, height, width of images and video).
//
// Queries are written rotated to their own tensor, keys rotated into the K
// cache and values as they are into the V cache: fp16 rows, or INT8 / INT4
// rows quantized per token from the fp16-rounded values, so the cache holds
// what rotating first and appending after would leave there.
//
// Bound by memory: every row is read and written once. One block holds 32 rows
// (heads) of 128 channels of a token, or of a few tokens, an 8-lane group each;
// its first threads work out the tokens' cosines and sines while the rows arrive.
// 8192 tokens of 32 + 8 + 8 heads into fp16 caches take 36 us (5.6 TB/s), 2047
// into INT8 14.3 us (7.1 of them for the bytes), where a row's maximum is waited for
// before its codes; 8 tokens 1.9 us on the GPU, less than their launch takes the host.
// Angles take a 64-bit product and range reduction: positions of 10^5 and more
// leave no correct digits in fp32 at the highest frequencies.
// Built with -fmad=false: the products round like separate operations.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "lik_device.cuh"
#include "lik_internal.h"
#include "lik_quant.cuh"

namespace lik {

namespace {

constexpr int kMaxFreqs = kHeadDim / 2;
constexpr int kRows = 32;   // rows of a block
constexpr int kTokens = 3;  // tokens of a block, where there are many

struct RopeParams {
    const __half* q;
    const __half* k;
    const __half* v;
    const long long* pos;  // [axes, n_tokens]
    const float* inv_freq;
    const long long* slots;
    __half* q_out;
    uint8_t* k_cache;
    uint8_t* v_cache;
    __half* k_scale;
    __half* v_scale;
    __half* v_zero;
    long long q_stride, k_stride, v_stride;  // elements between tokens
    long long n_tokens, n_slots;
    int n_heads, n_kv, block_size, freqs;
    int k_format, v_format;
    int section_end[4];
};

enum Pairs : int { kHalves = 0, kNeighbours = 1, kHalvesAny = 2 };

__device__ __forceinline__ void rotate2(uint32_t& x, uint32_t& y, float2 c0, float2 c1) {  // two (a, b) pairs
    const float2 a = __half22float2(as_h2(x)), b = __half22float2(as_h2(y));
    x = as_u32(__floats2half2_rn(__fsub_rn(__fmul_rn(a.x, c0.x), __fmul_rn(b.x, c0.y)),
                                 __fsub_rn(__fmul_rn(a.y, c1.x), __fmul_rn(b.y, c1.y))));
    y = as_u32(__floats2half2_rn(__fadd_rn(__fmul_rn(b.x, c0.x), __fmul_rn(a.x, c0.y)),
                                 __fadd_rn(__fmul_rn(b.y, c1.x), __fmul_rn(a.y, c1.y))));
}
__device__ __forceinline__ uint32_t rotate1(uint32_t x, float2 c) {  // one (a, b) pair
    const float2 a = __half22float2(as_h2(x));
    return as_u32(__floats2half2_rn(__fsub_rn(__fmul_rn(a.x, c.x), __fmul_rn(a.y, c.y)),
                                    __fadd_rn(__fmul_rn(a.y, c.x), __fmul_rn(a.x, c.y))));
}

__device__ __forceinline__ void store_cache_row(int format, const Raw16& raw, long long row, uint8_t* cache,
                                                __half* scale, __half* zero, int l, unsigned mask) {
    switch (format) {
        case kF16: {
            uint4* dst = reinterpret_cast<uint4*>(cache + row * (kHeadDim * 2)) + 2 * l;
            dst[0] = raw.a;
            dst[1] = raw.b;
            break;
        }
        case kI8: quant_row<kTokI8>(raw, row, cache, scale, zero, l, mask); break;
        case kI4Sym: quant_row<kTokI4Sym>(raw, row, cache, scale, zero, l, mask); break;
        default: quant_row<kTokI4Asym>(raw, row, cache, scale, zero, l, mask); break;
    }
}

// Where frequency f's cosine and sine lie: lane l reads those of 8 l .. 8 l + 7 two
// at a time, and the eight lanes' reads then fill one run of 128 bytes (8192
// tokens: 35.8 us; 39.3 with them in order, where half the banks' reads collided).
// kHalvesAny reads them one by one.
template <int PAIRS>
__device__ __forceinline__ int turn_at(int f) {
    return PAIRS == kHalvesAny ? f : (f & 6) * 8 + (f >> 3) * 2 + (f & 1);
}

// PAIRS kHalves: the frequencies fill whole 16-byte chunks (r a multiple of
// 8), so lane l < r / 8 holds chunks l and l + r / 8, both halves of its pairs;
// the other lanes hold the chunks that pass. kHalvesAny (any r) and
// kNeighbours: lane l holds channels 16 l .. 16 l + 15. A block takes TOK
// tokens, whose rows are all on their way before the first is used; more than
// one only where both caches are fp16.
template <int PAIRS, int TOK>
__global__ void __launch_bounds__(256, TOK == 1 ? 8 : 6) rope_append_kernel(const __grid_constant__ RopeParams p) {
    __shared__ __align__(16) float2 turn[TOK][kMaxFreqs];  // cosine, sine; see turn_at
    const long long tok0 = static_cast<long long>(blockIdx.x) * TOK;
    const int l = threadIdx.x & 7;
    const unsigned mask = 0xFFu << (threadIdx.x & 24);
    const int row = blockIdx.y * kRows + (threadIdx.x >> 3);
    const int kind = row < p.n_heads ? 0 : row < p.n_heads + p.n_kv ? 1 : 2;
    const bool here = row < p.n_heads + 2 * p.n_kv;
    const int head = kind == 0 ? row : row - p.n_heads - (kind == 2 ? p.n_kv : 0);
    const long long stride = kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride;
    const __half* src = (kind == 0 ? p.q : kind == 1 ? p.k : p.v) + tok0 * stride + static_cast<size_t>(head) * kHeadDim;
    const int c = p.freqs / 8;
    const int k_format = TOK == 1 ? p.k_format : kF16, v_format = TOK == 1 ? p.v_format : kF16;
    int x0 = 2 * l, x1 = 2 * l + 1;  // the 16-byte chunks this lane holds
    if (PAIRS == kHalves && kind != 2 && l < c) {
        x0 = l;
        x1 = l + c;
    }
    Raw16 rows[TOK];
#pragma unroll
    for (int t = 0; t < TOK; ++t) {
        if (here && tok0 + t < p.n_tokens) {
            rows[t].a = __ldcs(reinterpret_cast<const uint4*>(src + t * stride) + x0);
            rows[t].b = __ldcs(reinterpret_cast<const uint4*>(src + t * stride) + x1);
        }
    }
    if (threadIdx.x < TOK * kMaxFreqs) {
        const int t = threadIdx.x / kMaxFreqs, f = threadIdx.x % kMaxFreqs;
        if (f < p.freqs && tok0 + t < p.n_tokens) {
            const int axis = (f >= p.section_end[0]) + (f >= p.section_end[1]) + (f >= p.section_end[2]);
            constexpr double per_turn = 0.15915494309189533577;  // 1 / (2 pi)
            const double turns = static_cast<double>(p.pos[axis * p.n_tokens + tok0 + t]) *
                                 static_cast<double>(p.inv_freq[f]) * per_turn;
            float s, co;
            sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &co);
            turn[t][turn_at<PAIRS>(f)] = {co, s};
        }
    }
    __syncthreads();
    if (!here) return;  // whole 8-lane groups leave together
#pragma unroll
    for (int t = 0; t < TOK; ++t) {
        const long long tok = tok0 + t;
        if (tok >= p.n_tokens) return;
        Raw16 raw = rows[t];
        const float2* const cs = turn[t];
        if (kind != 2) {
            uint32_t* a = reinterpret_cast<uint32_t*>(&raw.a);
            uint32_t* b = reinterpret_cast<uint32_t*>(&raw.b);
            if (PAIRS == kHalves) {
                if (l < c) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 u = *reinterpret_cast<const float4*>(cs + turn_at<PAIRS>(8 * l + 2 * i));
                        rotate2(a[i], b[i], {u.x, u.y}, {u.z, u.w});
                    }
                }
            } else if (PAIRS == kNeighbours) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 u = *reinterpret_cast<const float4*>(cs + turn_at<PAIRS>(8 * l + 2 * i));
                    uint32_t& x = i < 2 ? a[2 * i] : b[2 * i - 4];
                    uint32_t& y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
                    if (8 * l + 2 * i < p.freqs) x = rotate1(x, {u.x, u.y});
                    if (8 * l + 2 * i + 1 < p.freqs) y = rotate1(y, {u.z, u.w});
                }
            } else {
                // a pair's other channel sits in another lane: read it once more
                const __half* row_at = src + t * stride;
                __half* h = reinterpret_cast<__half*>(&raw);
                if (16 * l < 2 * p.freqs) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int ch = 16 * l + i;
                        if (ch >= 2 * p.freqs) continue;
                        const bool first = ch < p.freqs;
                        const float x = __half2float(h[i]);
                        const float y = __half2float(row_at[first ? ch + p.freqs : ch - p.freqs]);
                        const float2 u = cs[turn_at<PAIRS>(first ? ch : ch - p.freqs)];
                        h[i] = __float2half_rn(first ? __fsub_rn(__fmul_rn(x, u.x), __fmul_rn(y, u.y))
                                                     : __fadd_rn(__fmul_rn(x, u.x), __fmul_rn(y, u.y)));
                    }
                }
                __syncwarp(mask);  // q may be rotated in place: nobody writes before all have read
            }
        }
        if (kind == 0) {
            uint4* dst = reinterpret_cast<uint4*>(p.q_out + (tok * p.n_heads + head) * kHeadDim);
            dst[x0] = raw.a;
            dst[x1] = raw.b;
            continue;
        }
        const long long slot = p.slots[tok];
        if (slot < 0 || slot >= p.n_slots) continue;  // a token that is not kept
        const long long blk = p.n_slots <= 0x7fffffffLL
                                  ? static_cast<long long>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.block_size))
                                  : slot / p.block_size;
        const long long drow = (blk * p.n_kv + head) * p.block_size + (slot - blk * p.block_size);
        if (kind == 2) {
            store_cache_row(v_format, raw, drow, p.v_cache, p.v_scale, p.v_zero, l, mask);
            continue;
        }
        if (PAIRS == kHalves && k_format != kF16) {
            // bring the row into 16 consecutive channels per lane: chunk x sits in
            // lane x (first half), x - c (second half) or x / 2 (passing chunks)
            const uint32_t a[4] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w}, b[4] = {raw.b.x, raw.b.y, raw.b.z, raw.b.w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int x = 2 * l + j;
                const int from = x < c ? x : x < 2 * c ? x - c : x >> 1;
                const bool second = x < c ? false : x < 2 * c ? true : (x & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t u = __shfl_sync(mask, a[i], from, 8), w = __shfl_sync(mask, b[i], from, 8);
                    o[4 * j + i] = second ? w : u;
                }
            }
            raw.a = {o[0], o[1], o[2], o[3]};
            raw.b = {o[4], o[5], o[6], o[7]};
        } else if (PAIRS == kHalves) {
            uint4* dst = reinterpret_cast<uint4*>(p.k_cache + drow * (kHeadDim * 2));
            dst[x0] = raw.a;
            dst[x1] = raw.b;
            continue;
        }
        store_cache_row(k_format, raw, drow, p.k_cache, p.k_scale, nullptr, l, mask);
    }
}

template <int PAIRS, int TOK>
void launch_tokens(const RopeParams& p, cudaStream_t stream) {
    const unsigned rows = static_cast<unsigned>((p.n_heads + 2 * p.n_kv + kRows - 1) / kRows);
    const unsigned blocks = static_cast<unsigned>((p.n_tokens + TOK - 1) / TOK);
    rope_append_kernel<PAIRS, TOK><<<dim3(blocks, rows), 256, 0, stream>>>(p);
}

// kTokens tokens per block keep more rows in flight. It pays where the work is
// copying and there are tokens enough for every SM: 32 + 8 + 8 heads, fp16
// caches, 35.3 instead of 37.3 us for 8000 tokens, 17.3 instead of 18.8 for
// 4000, the same for 2000 and fewer. Two tokens were slower (36.0), and four for
// 4000 tokens (18.8). Rows that are quantized wait for their reductions, one token
// after the other: 8000 tokens into INT8 took 76 us with four tokens per block
// and 67 with one (55.9 with the registers held to 32, eight blocks on an SM), a
// dequantizing call of 13 us beside it included; the append alone takes 42.8.
template <int PAIRS>
void launch_pairs(const RopeParams& p, cudaStream_t stream, int sm_count) {
    const long long rows = p.n_tokens * (p.n_heads + 2 * p.n_kv);
    if (p.k_format == kF16 && p.v_format == kF16 && rows >= 1024LL * sm_count)
        launch_tokens<PAIRS, kTokens>(p, stream);
    else
        launch_tokens<PAIRS, 1>(p, stream);
}

}  // namespace

lik_status launch_rope_append(const RopeAppendArgs& a, cudaStream_t stream, std::string& err) {
    RopeParams p{};
    p.q = static_cast<const __half*>(a.q);
    p.k = static_cast<const __half*>(a.k);
    p.v = static_cast<const __half*>(a.v);
    p.pos = reinterpret_cast<const long long*>(a.positions);
    p.inv_freq = a.inv_freq;
    p.slots = reinterpret_cast<const long long*>(a.slot_mapping);
    p.q_out = static_cast<__half*>(a.q_out);
    p.k_cache = static_cast<uint8_t*>(a.k_cache);
    p.v_cache = static_cast<uint8_t*>(a.v_cache);
    p.k_scale = static_cast<__half*>(a.k_scale);
    p.v_scale = static_cast<__half*>(a.v_scale);
    p.v_zero = static_cast<__half*>(a.v_zero);
    p.q_stride = a.q_token_stride;
    p.k_stride = a.k_token_stride;
    p.v_stride = a.v_token_stride;
    p.n_tokens = a.n_tokens;
    p.n_slots = a.num_blocks * a.block_size;
    p.n_heads = static_cast<int>(a.n_heads);
    p.n_kv = static_cast<int>(a.n_kv_heads);
    p.block_size = static_cast<int>(a.block_size);
    p.freqs = static_cast<int>(a.n_freqs);
    p.k_format = a.k_format;
    p.v_format = a.v_format;
    int end = 0;
    for (int i = 0; i < 4; ++i) {
        end = i < a.n_axes - 1 ? end + static_cast<int>(a.sections[i]) : kMaxFreqs;
        p.section_end[i] = end;
    }
    DeviceInfo di;
    if (!device_info(di, err)) return LIK_ERR_CUDA;
    if (a.interleaved)
        launch_pairs<kNeighbours>(p, stream, di.sm_count);
    else if (p.freqs % 8 == 0)
        launch_pairs<kHalves>(p, stream, di.sm_count);
    else
        launch_tokens<kHalvesAny, 1>(p, stream);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        err = std::string("rotating append launch: ") + cudaGetErrorString(e);
        return LIK_ERR_CUDA;
    }
    return LIK_OK;
}

}  // namespace lik
