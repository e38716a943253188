// KV quantize / pack kernels for sm_100a, bit-exact with the reference's
// PyTorch oracle (reference/kv_cache_ref.py:46-62, 73-112) on fp16 inputs
// viewed as fp32:
//   scale = max(absmax / qmax, 1e-8)        IEEE fp32 division
//   code  = clamp(rint(x / scale), +-qmax)  IEEE division, round half to even
//   stored scale = fp16(scale)              round to nearest even
// This translation unit is compiled without --use_fast_math and with
// -fmad=false; divisions go through __fdiv_rn explicitly.
//
// The reference CUDA kernels (kernels/kv_cache/kv_compress.cu) multiply by a
// reciprocal instead and differ from the oracle by one code at ~6e-5 of
// positions; these kernels do not.
//
// Every kernel writes into a destination cache of allocated length
// dst_buf_len at position dst_pos, so the same code serves the reference's
// one-shot ops (dst_pos = 0, dst_buf_len = n_tokens) and in-place append into a
// preallocated cache.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "lik_device.cuh"
#include "lik_internal.h"
#include "lik_quant.cuh"

namespace lik {

namespace {

template <int MODE>
__global__ void __launch_bounds__(256, 4) quant_token_kernel(const __half* __restrict__ x, uint8_t* __restrict__ codes,
                                                          __half* __restrict__ scale, __half* __restrict__ zero,
                                                          long long n_rows, long long n_tok, long long dst_pos,
                                                          long long dst_buf) {
    constexpr int R = kRowsPerGroup;
    constexpr int NL = kLanesPerRow;
    constexpr int CH = kHeadDim / NL;  // channels per lane
    const long long row0 = ((static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / NL) * R;
    if (row0 >= n_rows) return;  // whole 8-lane groups leave together
    const int l = threadIdx.x & (NL - 1);
    const unsigned mask = 0xFFu << (threadIdx.x & 24);
    Raw16 raw[R];
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (row0 + k < n_rows) raw[k] = load_raw16(x + (row0 + k) * kHeadDim + l * CH);

    long long slab = row0 / n_tok;
    long long t = row0 - slab * n_tok;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        if (row0 + k >= n_rows) break;  // the same for the whole 8-lane group
        const long long drow = slab * dst_buf + dst_pos + t;
        if (++t == n_tok) {
            t = 0;
            ++slab;
        }
        quant_row<MODE>(raw[k], drow, codes, scale, zero, l, mask);
    }
}

// ---- per-token quantize of a whole tensor: 4 lanes per row -----------------
// Each row is held by 4 lanes (32 channels, 64 bytes each), so the per-row
// work (statistics, scale, reciprocal) is shared by 128 elements per lane
// quartet; the grid is persistent and every lane quartet prefetches its next
// row while it quantizes the current one. Same arithmetic as quant_row.

// Division of 32-bit row indices by a launch constant with one multiply-high
// (the round-up method of Granlund and Montgomery): q = (umulhi(x, m) + x) >> s.
struct RowDiv {
    uint32_t d, m, s;
    __device__ __forceinline__ uint32_t q(uint32_t x) const { return (__umulhi(x, m) + x) >> s; }
};
RowDiv make_rowdiv(uint32_t d) {
    RowDiv f{d, 0u, 0u};
    while ((uint64_t{1} << f.s) < d) ++f.s;
    f.m = static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << f.s) - d)) / d + 1);
    return f;
}

struct Raw32 {
    uint4 v[4];
};

// bytes b0..b3 of the result = (c[2i] & 0xF) | (c[2i+1] & 0xF) << 4
__device__ __forceinline__ uint32_t pack_nibbles8(const uint32_t* c) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = (c[2 * i] & 0xFu) | ((c[2 * i + 1] << 4) & 0xF0u);
    return pack_bytes4(b[0], b[1], b[2], b[3]);
}

template <int MODE>
__device__ __forceinline__ void quant_row32(const Raw32& raw, long long drow, uint8_t* __restrict__ codes,
                                            __half* __restrict__ scale, __half* __restrict__ zero, int l,
                                            unsigned mask) {
    const __half2* h = reinterpret_cast<const __half2*>(raw.v);  // 16 pairs
    float sf, zf = 0.f;
    if (MODE == kTokI4Asym) {
        __half2 mn2 = h[0], mx2 = h[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            mn2 = __hmin2(mn2, h[i]);
            mx2 = __hmax2(mx2, h[i]);
        }
        float mn = fminf(__low2float(mn2), __high2float(mn2));
        float mx = fmaxf(__low2float(mx2), __high2float(mx2));
#pragma unroll
        for (int m = 1; m < 4; m <<= 1) {
            mn = fminf(mn, __shfl_xor_sync(mask, mn, m));
            mx = fmaxf(mx, __shfl_xor_sync(mask, mx, m));
        }
        const float sc = fmaxf(__fdiv_rn(__fsub_rn(mx, mn), 15.0f), kAsymScaleFloor);
        const __half sh = __float2half_rn(sc);
        const __half zh = __float2half_rn(mn);
        sf = __half2float(sh);
        zf = __half2float(zh);
        if (l == 0) {
            scale[drow] = sh;
            zero[drow] = zh;
        }
    } else {
        constexpr float qmax = (MODE == kTokI8) ? 127.0f : 7.0f;
        __half2 am2 = __habs2(h[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) am2 = __hmax2(am2, __habs2(h[i]));
        float amax = fmaxf(__low2float(am2), __high2float(am2));
#pragma unroll
        for (int m = 1; m < 4; m <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, m));
        sf = fmaxf(__fdiv_rn(amax, qmax), 1e-8f);
        if (l == 0) scale[drow] = __float2half_rn(sf);
    }
    const float rf = __frcp_rn(sf);
    constexpr float lo = MODE == kTokI4Asym ? 0.0f : (MODE == kTokI8 ? -127.0f : -7.0f);
    constexpr float hi = MODE == kTokI4Asym ? 15.0f : (MODE == kTokI8 ? 127.0f : 7.0f);
#pragma unroll
    for (int ck = 0; ck < 2; ++ck) {  // 16 channels at a time
        float xv[16], tv[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 u = __half22float2(h[8 * ck + i]);
            xv[2 * i] = MODE == kTokI4Asym ? __fsub_rn(u.x, zf) : u.x;
            xv[2 * i + 1] = MODE == kTokI4Asym ? __fsub_rn(u.y, zf) : u.y;
        }
        bool exact = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = __fmul_rn(xv[i], rf);
            float tt = __fadd_rn(y, kRoundMagic);
            exact |= !(fabsf(__fsub_rn(y, __fsub_rn(tt, kRoundMagic))) < kNearTie);
            if (MODE == kTokI4Asym) tt = fminf(fmaxf(tt, kRoundMagic), kRoundMagic + 15.0f);
            tv[i] = tt;
        }
        if (exact) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                tv[i] = __fadd_rn(fminf(fmaxf(rintf(__fdiv_rn(xv[i], sf)), lo), hi), kRoundMagic);
        }
        uint32_t c[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = static_cast<uint32_t>(__float_as_int(tv[i]));
        if (MODE == kTokI8) {
            reinterpret_cast<uint4*>(codes + drow * kHeadDim + l * 32)[ck] =
                make_uint4(pack_bytes4(c[0], c[1], c[2], c[3]), pack_bytes4(c[4], c[5], c[6], c[7]),
                           pack_bytes4(c[8], c[9], c[10], c[11]), pack_bytes4(c[12], c[13], c[14], c[15]));
        } else {
            reinterpret_cast<uint2*>(codes + drow * (kHeadDim / 2) + l * 16)[ck] =
                make_uint2(pack_nibbles8(c), pack_nibbles8(c + 8));
        }
    }
}

template <int MODE>
__global__ void __launch_bounds__(256, 3) quant_rows_kernel(const __half* __restrict__ x, uint8_t* __restrict__ codes,
                                                         __half* __restrict__ scale, __half* __restrict__ zero,
                                                         uint32_t n_rows, RowDiv per_slab, long long dst_pos,
                                                         long long dst_buf) {
    const int l = threadIdx.x & 3;
    const unsigned mask = 0xFu << (threadIdx.x & 28);
    const uint32_t stride = (gridDim.x * blockDim.x) >> 2;
    uint32_t row = (blockIdx.x * blockDim.x + threadIdx.x) >> 2;
    if (row >= n_rows) return;  // whole lane quartets leave together
    auto load = [&](uint32_t rw) {
        Raw32 r;
        const uint4* src = reinterpret_cast<const uint4*>(x + static_cast<long long>(rw) * kHeadDim + l * 32);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.v[j] = __ldcs(src + j);
        return r;
    };
    auto quant = [&](const Raw32& r, uint32_t rw) {
        const uint32_t slab = per_slab.q(rw);
        const long long t = rw - slab * per_slab.d;
        quant_row32<MODE>(r, static_cast<long long>(slab) * dst_buf + dst_pos + t, codes, scale, zero, l, mask);
    };
    // two rows in flight, in alternating register sets
    Raw32 a = load(row), b = a;
    while (true) {
        const uint32_t r1 = row + stride;
        if (r1 < n_rows) b = load(r1);
        quant(a, row);
        if (r1 >= n_rows) break;
        const uint32_t r2 = r1 + stride;
        if (r2 < n_rows) a = load(r2);
        quant(b, r1);
        if (r2 >= n_rows) break;
        row = r2;
    }
}

// Append of new tokens into a paged cache [num_blocks, n_heads, block_size,
// row]: source rows are (token, kv head) of x [n_tokens, n_heads, 128]; token
// i goes to slot slots[i] = block * block_size + offset (slots < 0 or past the
// cache are skipped). MODE kAppendF16 copies fp16 rows; the others quantize
// per token like quant_token_kernel.
constexpr int kAppendF16 = -1;
template <int MODE>
__global__ void __launch_bounds__(256, 4) paged_append_kernel(const __half* __restrict__ x,
                                                           const long long* __restrict__ slots, long long n_rows,
                                                           int n_heads, int block_size, long long n_slots,
                                                           uint8_t* __restrict__ codes, __half* __restrict__ scale,
                                                           __half* __restrict__ zero) {
    constexpr int R = kRowsPerGroup;
    constexpr int NL = kLanesPerRow;
    constexpr int CH = kHeadDim / NL;
    const long long row0 = ((static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / NL) * R;
    if (row0 >= n_rows) return;
    const int l = threadIdx.x & (NL - 1);
    const unsigned mask = 0xFFu << (threadIdx.x & 24);
    Raw16 raw[R];
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (row0 + k < n_rows) raw[k] = load_raw16(x + (row0 + k) * kHeadDim + l * CH);
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const long long row = row0 + k;
        if (row >= n_rows) break;  // the same for the whole 8-lane group
        const long long tok = row / n_heads;
        const int h = static_cast<int>(row - tok * n_heads);
        const long long slot = slots[tok];
        if (slot < 0 || slot >= n_slots) continue;
        const long long blk = slot / block_size;
        const long long drow = (blk * n_heads + h) * block_size + (slot - blk * block_size);
        if (MODE == kAppendF16) {
            uint4* dst = reinterpret_cast<uint4*>(codes + drow * (kHeadDim * 2)) + 2 * l;
            dst[0] = raw[k].a;
            dst[1] = raw[k].b;
        } else {
            quant_row<MODE < 0 ? 0 : MODE>(raw[k], drow, codes, scale, zero, l, mask);
        }
    }
}

// Eight K channels of one token to packed nibbles, with the channels'
// scale, zero and reciprocal scale (the token kernels' rounding scheme).
template <bool ASYM>
__device__ __forceinline__ uint32_t quant8_k(const uint4& raw, const float (&sc)[8], const float (&zc)[8],
                                             const float (&rc)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
    float xv[8], tv[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = __half22float2(h[i]);
        xv[2 * i] = ASYM ? __fsub_rn(u.x, zc[2 * i]) : u.x;
        xv[2 * i + 1] = ASYM ? __fsub_rn(u.y, zc[2 * i + 1]) : u.y;
    }
    bool exact = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = __fmul_rn(xv[i], rc[i]);
        float tt = __fadd_rn(y, kRoundMagic);
        exact |= !(fabsf(__fsub_rn(y, __fsub_rn(tt, kRoundMagic))) < kNearTie);
        // asymmetric codes need the clamp (the zero point is rounded to fp16);
        // symmetric ones cannot leave [-7, 7]: |x| <= absmax <= 7 s (1 + 2^-24)
        if (ASYM) tt = fminf(fmaxf(tt, kRoundMagic), kRoundMagic + 15.0f);
        tv[i] = tt;
    }
    if (exact) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float qv = fminf(fmaxf(rintf(__fdiv_rn(xv[i], sc[i])), ASYM ? 0.0f : -7.0f), ASYM ? 15.0f : 7.0f);
            tv[i] = __fadd_rn(qv, kRoundMagic);
        }
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (static_cast<uint32_t>(__float_as_int(tv[i])) & 0xFu) << (4 * i);
    return w;
}

// One CTA per (slab, token group): 16 channel chunks x 16 token lanes.
// Pass 1 reduces each channel over the group's tokens (on packed fp16: min,
// max and |x| are exact); pass 2 writes packed codes. Groups of up to 128
// tokens stay in registers between the passes; longer groups are re-read.
// (register caps measured best on B200: 3 CTAs per SM with zero points, 4 without)
template <bool ASYM>
__global__ void __launch_bounds__(256, ASYM ? 3 : 4) quant_kgroup_kernel(const __half* __restrict__ x, uint8_t* __restrict__ codes,
                                                           __half* __restrict__ scale, __half* __restrict__ zero,
                                                           long long n_groups_new, long long n_tok, int gs,
                                                           long long dst_pos, long long dst_buf, long long ng_buf) {
    constexpr int MAXR = 8;  // token rows a thread keeps in registers
    __shared__ float red_a[16][kHeadDim];
    __shared__ float red_b[16][kHeadDim];
    __shared__ float s_scale[kHeadDim];
    __shared__ float s_zero[kHeadDim];
    __shared__ float s_rcp[kHeadDim];

    const long long blk = blockIdx.x;
    const long long slab = blk / n_groups_new;
    const long long g = blk - slab * n_groups_new;
    const int cc = threadIdx.x & 15;
    const int tl = threadIdx.x >> 4;
    const long long t0 = g * gs;
    const long long t1 = min(t0 + gs, n_tok);
    const __half* xs = x + slab * n_tok * kHeadDim + cc * 8;
    const bool in_regs = (t1 - t0) <= 16 * MAXR;  // the same for the whole CTA

    const uint32_t pinf = 0x7C007C00u, ninf = 0xFC00FC00u;
    __half2 a2[4], b2[4];  // per channel pair: min (asym) or absmax (sym); max (asym)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a2[i] = ASYM ? *reinterpret_cast<const __half2*>(&pinf) : __float2half2_rn(0.0f);
        b2[i] = *reinterpret_cast<const __half2*>(&ninf);
    }
    auto stats = [&](const uint4& raw) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (ASYM) {
                a2[i] = __hmin2(a2[i], h[i]);
                b2[i] = __hmax2(b2[i], h[i]);
            } else {
                a2[i] = __hmax2(a2[i], __habs2(h[i]));
            }
        }
    };
    uint4 raw[MAXR];
    if (in_regs) {
#pragma unroll
        for (int r = 0; r < MAXR; ++r) {
            const long long t = t0 + tl + 16 * r;
            if (t < t1) raw[r] = *reinterpret_cast<const uint4*>(xs + t * kHeadDim);
        }
#pragma unroll
        for (int r = 0; r < MAXR; ++r)
            if (t0 + tl + 16 * r < t1) stats(raw[r]);
    } else {
        for (long long t = t0 + tl; t < t1; t += 16) stats(*reinterpret_cast<const uint4*>(xs + t * kHeadDim));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        red_a[tl][cc * 8 + 2 * i] = __low2float(a2[i]);
        red_a[tl][cc * 8 + 2 * i + 1] = __high2float(a2[i]);
        if (ASYM) {
            red_b[tl][cc * 8 + 2 * i] = __low2float(b2[i]);
            red_b[tl][cc * 8 + 2 * i + 1] = __high2float(b2[i]);
        }
    }
    __syncthreads();
    if (threadIdx.x < kHeadDim) {
        const int ch = threadIdx.x;
        float ra = red_a[0][ch], rb = ASYM ? red_b[0][ch] : 0.0f;
        for (int r = 1; r < 16; ++r) {
            if (ASYM) {
                ra = fminf(ra, red_a[r][ch]);
                rb = fmaxf(rb, red_b[r][ch]);
            } else {
                ra = fmaxf(ra, red_a[r][ch]);
            }
        }
        const long long gidx = (slab * ng_buf + dst_pos / gs + g) * kHeadDim + ch;
        if (ASYM) {
            const float s = fmaxf(__fdiv_rn(__fsub_rn(rb, ra), 15.0f), kAsymScaleFloor);
            const __half sh = __float2half_rn(s);
            const __half zh = __float2half_rn(ra);
            s_scale[ch] = __half2float(sh);
            s_zero[ch] = __half2float(zh);
            s_rcp[ch] = __frcp_rn(__half2float(sh));
            scale[gidx] = sh;
            zero[gidx] = zh;
        } else {
            const float s = fmaxf(__fdiv_rn(ra, 7.0f), 1e-8f);
            s_scale[ch] = s;
            s_rcp[ch] = __frcp_rn(s);
            scale[gidx] = __float2half_rn(s);
        }
    }
    __syncthreads();
    float sc[8], zc[8], rc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sc[i] = s_scale[cc * 8 + i];
        zc[i] = ASYM ? s_zero[cc * 8 + i] : 0.0f;
        rc[i] = s_rcp[cc * 8 + i];
    }
    uint8_t* dst = codes + (slab * dst_buf + dst_pos) * (kHeadDim / 2);
    if (in_regs) {
#pragma unroll
        for (int r = 0; r < MAXR; ++r) {
            const long long t = t0 + tl + 16 * r;
            if (t < t1) reinterpret_cast<uint32_t*>(dst + t * (kHeadDim / 2))[cc] = quant8_k<ASYM>(raw[r], sc, zc, rc);
        }
    } else {
        for (long long t = t0 + tl; t < t1; t += 16)
            reinterpret_cast<uint32_t*>(dst + t * (kHeadDim / 2))[cc] =
                quant8_k<ASYM>(*reinterpret_cast<const uint4*>(xs + t * kHeadDim), sc, zc, rc);
    }
}

}  // namespace

lik_status launch_quant_token(int mode, const void* x, void* codes, void* scale, void* zero, int64_t n_slabs,
                              int64_t n_tokens, int64_t dst_pos, int64_t dst_buf_len, cudaStream_t stream,
                              std::string& err) {
    const long long n_rows = static_cast<long long>(n_slabs) * n_tokens;
    if (n_rows == 0) return LIK_OK;
    const long long rows_per_block = (256LL / kLanesPerRow) * kRowsPerGroup;
    const long long blocks = (n_rows + rows_per_block - 1) / rows_per_block;
    if (blocks > 0x7fffffffLL) {
        err = "too many rows";
        return LIK_ERR_INVALID_ARGUMENT;
    }
    const __half* xh = static_cast<const __half*>(x);
    uint8_t* c = static_cast<uint8_t*>(codes);
    __half* s = static_cast<__half*>(scale);
    __half* z = static_cast<__half*>(zero);
    DeviceInfo di;
    if (n_rows < (1LL << 31) && n_tokens > 0 && device_info(di, err)) {
        const long long need = (n_rows + 63) / 64;  // 64 rows per 256-thread block
        const unsigned nb = static_cast<unsigned>(std::min<long long>(need, 3LL * di.sm_count));
        const RowDiv per_slab = make_rowdiv(static_cast<uint32_t>(n_tokens));
        const uint32_t nr = static_cast<uint32_t>(n_rows);
        switch (mode) {
            case kTokI8: quant_rows_kernel<kTokI8><<<nb, 256, 0, stream>>>(xh, c, s, z, nr, per_slab, dst_pos, dst_buf_len); break;
            case kTokI4Sym: quant_rows_kernel<kTokI4Sym><<<nb, 256, 0, stream>>>(xh, c, s, z, nr, per_slab, dst_pos, dst_buf_len); break;
            default: quant_rows_kernel<kTokI4Asym><<<nb, 256, 0, stream>>>(xh, c, s, z, nr, per_slab, dst_pos, dst_buf_len); break;
        }
    } else switch (mode) {
        case kTokI8:
            quant_token_kernel<kTokI8><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(xh, c, s, z, n_rows, n_tokens,
                                                                                         dst_pos, dst_buf_len);
            break;
        case kTokI4Sym:
            quant_token_kernel<kTokI4Sym><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
                xh, c, s, z, n_rows, n_tokens, dst_pos, dst_buf_len);
            break;
        default:
            quant_token_kernel<kTokI4Asym><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
                xh, c, s, z, n_rows, n_tokens, dst_pos, dst_buf_len);
            break;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        err = std::string("quantize launch: ") + cudaGetErrorString(e);
        return LIK_ERR_CUDA;
    }
    return LIK_OK;
}

lik_status launch_paged_append(int row_format, const void* x, const int64_t* slots, int64_t n_tokens,
                               int64_t n_heads, void* cache, void* scale, void* zero, int64_t num_blocks,
                               int64_t block_size, cudaStream_t stream, std::string& err) {
    const long long n_rows = static_cast<long long>(n_tokens) * n_heads;
    if (n_rows == 0) return LIK_OK;
    const long long rows_per_block = (256LL / kLanesPerRow) * kRowsPerGroup;
    const long long blocks = (n_rows + rows_per_block - 1) / rows_per_block;
    if (blocks > 0x7fffffffLL) {
        err = "too many rows";
        return LIK_ERR_INVALID_ARGUMENT;
    }
    const __half* xh = static_cast<const __half*>(x);
    const long long* sl = reinterpret_cast<const long long*>(slots);
    uint8_t* c = static_cast<uint8_t*>(cache);
    __half* s = static_cast<__half*>(scale);
    __half* z = static_cast<__half*>(zero);
    const long long n_slots = static_cast<long long>(num_blocks) * block_size;
    const unsigned nb = static_cast<unsigned>(blocks);
    const int nh = static_cast<int>(n_heads), bs = static_cast<int>(block_size);
    switch (row_format) {
        case 0: paged_append_kernel<kAppendF16><<<nb, 256, 0, stream>>>(xh, sl, n_rows, nh, bs, n_slots, c, s, z); break;
        case 1: paged_append_kernel<kTokI8><<<nb, 256, 0, stream>>>(xh, sl, n_rows, nh, bs, n_slots, c, s, z); break;
        case 2: paged_append_kernel<kTokI4Sym><<<nb, 256, 0, stream>>>(xh, sl, n_rows, nh, bs, n_slots, c, s, z); break;
        default: paged_append_kernel<kTokI4Asym><<<nb, 256, 0, stream>>>(xh, sl, n_rows, nh, bs, n_slots, c, s, z); break;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        err = std::string("paged append launch: ") + cudaGetErrorString(e);
        return LIK_ERR_CUDA;
    }
    return LIK_OK;
}

lik_status launch_quant_kgroup(bool asym, const void* x, void* codes, void* scale, void* zero, int64_t n_slabs,
                               int64_t n_tokens, int64_t group_size, int64_t dst_pos, int64_t dst_buf_len,
                               int64_t n_groups_buf, cudaStream_t stream, std::string& err) {
    const long long ngn = (n_tokens + group_size - 1) / group_size;
    const long long blocks = static_cast<long long>(n_slabs) * ngn;
    if (blocks == 0) return LIK_OK;
    if (blocks > 0x7fffffffLL) {
        err = "too many groups";
        return LIK_ERR_INVALID_ARGUMENT;
    }
    const __half* xh = static_cast<const __half*>(x);
    uint8_t* c = static_cast<uint8_t*>(codes);
    __half* s = static_cast<__half*>(scale);
    __half* z = static_cast<__half*>(zero);
    if (asym) {
        quant_kgroup_kernel<true><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
            xh, c, s, z, ngn, n_tokens, static_cast<int>(group_size), dst_pos, dst_buf_len, n_groups_buf);
    } else {
        quant_kgroup_kernel<false><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
            xh, c, s, z, ngn, n_tokens, static_cast<int>(group_size), dst_pos, dst_buf_len, n_groups_buf);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        err = std::string("quantize launch: ") + cudaGetErrorString(e);
        return LIK_ERR_CUDA;
    }
    return LIK_OK;
}

}  // namespace lik

// ---- dequantize to fp16 (prefill / materialize path) -----------------------
// fp16(code * scale [+ zero]) exactly as the reference's dequantize helpers
// compute it (fp32 product, one rounding to fp16; the asymmetric add happens in
// fp32 before the rounding). One 16-lane half-warp per token row.

namespace lik {
namespace {

// Packed fp32 pair arithmetic (sm_100: one instruction for two IEEE
// round-to-nearest results, the same values as two scalar operations).
__device__ __forceinline__ float2 mul2_rn(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2_rn(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// FMT: 0 = INT8 per token, 1 = INT4 KIVI symmetric, 2 = INT4 KIVI asymmetric.
template <int FMT>
__device__ __forceinline__ void dequant_row(const uint8_t* __restrict__ kq, const __half* __restrict__ ks,
                                            const __half* __restrict__ kz, const uint8_t* __restrict__ vq,
                                            const __half* __restrict__ vs, const __half* __restrict__ vz,
                                            __half* __restrict__ kout, __half* __restrict__ vout, long long row,
                                            long long seqlen, long long buf, int gs, long long ng_buf, int scale_vec,
                                            int l) {
    const long long slab = row / seqlen;
    const long long t = row - slab * seqlen;
    const long long src = slab * buf + t;
    if (FMT == 0) {
        float k[8], v[8];
        const uint2 a = reinterpret_cast<const uint2*>(kq + src * kHeadDim)[l];
        const uint2 b = reinterpret_cast<const uint2*>(vq + src * kHeadDim)[l];
        const float sk = __half2float(ks[src]), sv = __half2float(vs[src]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k[i] = static_cast<float>(static_cast<int8_t>(a.x >> (8 * i))) * sk;
            k[4 + i] = static_cast<float>(static_cast<int8_t>(a.y >> (8 * i))) * sk;
            v[i] = static_cast<float>(static_cast<int8_t>(b.x >> (8 * i))) * sv;
            v[4 + i] = static_cast<float>(static_cast<int8_t>(b.y >> (8 * i))) * sv;
        }
        uint4 ko, vo;
        __half* kh = reinterpret_cast<__half*>(&ko);
        __half* vh = reinterpret_cast<__half*>(&vo);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            kh[i] = __float2half_rn(k[i]);
            vh[i] = __float2half_rn(v[i]);
        }
        reinterpret_cast<uint4*>(kout + row * kHeadDim)[l] = ko;
        reinterpret_cast<uint4*>(vout + row * kHeadDim)[l] = vo;
    } else {
        const uint32_t a = reinterpret_cast<const uint32_t*>(kq + src * (kHeadDim / 2))[l];
        const uint32_t b = reinterpret_cast<const uint32_t*>(vq + src * (kHeadDim / 2))[l];
        const long long g = slab * ng_buf + t / gs;
        const float sv = __half2float(vs[src]);
        const float zv = FMT == 2 ? __half2float(vz[src]) : 0.f;
        // the lane's 8 K group scales (and zeros): one 16-byte load each when
        // the scale tensors are 16-byte aligned, else eight 2-byte loads
        uint4 ksv, kzv = make_uint4(0, 0, 0, 0);
        __half* ksw = reinterpret_cast<__half*>(&ksv);
        __half* kzw = reinterpret_cast<__half*>(&kzv);
        if (scale_vec) {
            ksv = reinterpret_cast<const uint4*>(ks + g * kHeadDim)[l];
            if (FMT == 2) kzv = reinterpret_cast<const uint4*>(kz + g * kHeadDim)[l];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ksw[i] = ks[g * kHeadDim + 8 * l + i];
                if (FMT == 2) kzw[i] = kz[g * kHeadDim + 8 * l + i];
            }
        }
        // nibbles -> exact floats: OR each into the mantissa of 1.5 * 2^23
        // and subtract (signed nibbles offset by 8 first); then, per channel
        // pair, fp32 code * scale (+ zero) with the oracle's roundings and one
        // rounding to fp16
        constexpr uint32_t kFlip = FMT == 1 ? 0x88888888u : 0u;
        constexpr float kBase = FMT == 1 ? 12582920.0f : 12582912.0f;  // 1.5 * 2^23 (+ 8)
        const uint32_t af = a ^ kFlip, bf = b ^ kFlip;
        const __half2* ks2 = reinterpret_cast<const __half2*>(&ksv);
        const __half2* kz2 = reinterpret_cast<const __half2*>(&kzv);
        const float2 base = make_float2(kBase, kBase);
        const float2 sv2 = make_float2(sv, sv), zv2 = make_float2(zv, zv);
        uint4 ko, vo;
        uint32_t* kw = reinterpret_cast<uint32_t*>(&ko);
        uint32_t* vw = reinterpret_cast<uint32_t*>(&vo);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 ck = add2_rn(make_float2(__uint_as_float(0x4B400000u | ((af >> (8 * i)) & 0xFu)),
                                                  __uint_as_float(0x4B400000u | ((af >> (8 * i + 4)) & 0xFu))),
                                      make_float2(-base.x, -base.y));
            const float2 cv = add2_rn(make_float2(__uint_as_float(0x4B400000u | ((bf >> (8 * i)) & 0xFu)),
                                                  __uint_as_float(0x4B400000u | ((bf >> (8 * i + 4)) & 0xFu))),
                                      make_float2(-base.x, -base.y));
            float2 kf = mul2_rn(ck, __half22float2(ks2[i]));
            float2 vf = mul2_rn(cv, sv2);
            if (FMT == 2) {
                kf = add2_rn(kf, __half22float2(kz2[i]));
                vf = add2_rn(vf, zv2);
            }
            const __half2 kh2 = __floats2half2_rn(kf.x, kf.y);
            const __half2 vh2 = __floats2half2_rn(vf.x, vf.y);
            kw[i] = *reinterpret_cast<const uint32_t*>(&kh2);
            vw[i] = *reinterpret_cast<const uint32_t*>(&vh2);
        }
        reinterpret_cast<uint4*>(kout + row * kHeadDim)[l] = ko;
        reinterpret_cast<uint4*>(vout + row * kHeadDim)[l] = vo;
    }
}

// One 16-lane half-warp per two consecutive token rows (8 channels per lane
// and row), so that each lane has both rows' loads in flight.
constexpr int kDequantRows = 2;
template <int FMT>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* __restrict__ kq, const __half* __restrict__ ks,
                                                     const __half* __restrict__ kz, const uint8_t* __restrict__ vq,
                                                     const __half* __restrict__ vs, const __half* __restrict__ vz,
                                                     __half* __restrict__ kout, __half* __restrict__ vout,
                                                     long long n_rows, long long seqlen, long long buf, int gs,
                                                     long long ng_buf, int scale_vec) {
    const long long row0 = ((static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4) * kDequantRows;
    const int l = threadIdx.x & 15;
#pragma unroll
    for (int k = 0; k < kDequantRows; ++k)
        if (row0 + k < n_rows)
            dequant_row<FMT>(kq, ks, kz, vq, vs, vz, kout, vout, row0 + k, seqlen, buf, gs, ng_buf, scale_vec, l);
}

}  // namespace

lik_status launch_dequant(int fmt, const void* kq, const void* ks, const void* kz, const void* vq, const void* vs,
                          const void* vz, void* kout, void* vout, int64_t n_slabs, int64_t seqlen,
                          int64_t kv_buf_len, int64_t group_size, int64_t n_groups_buf, cudaStream_t stream,
                          std::string& err) {
    const long long n_rows = static_cast<long long>(n_slabs) * seqlen;
    if (n_rows == 0) return LIK_OK;
    const long long blocks = (n_rows + 16 * kDequantRows - 1) / (16 * kDequantRows);
    if (blocks > 0x7fffffffLL) {
        err = "too many rows";
        return LIK_ERR_INVALID_ARGUMENT;
    }
    auto c = [](const void* p) { return static_cast<const uint8_t*>(p); };
    auto h = [](const void* p) { return static_cast<const __half*>(p); };
    __half* ko = static_cast<__half*>(kout);
    __half* vo = static_cast<__half*>(vout);
    const int gs = static_cast<int>(group_size > 0 ? group_size : 1);
    const unsigned nb = static_cast<unsigned>(blocks);
    auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
    const int vec = (fmt != 0 && al16(ks) && (fmt != 2 || al16(kz))) ? 1 : 0;
    if (fmt == 0)
        dequant_kernel<0><<<nb, 256, 0, stream>>>(c(kq), h(ks), h(kz), c(vq), h(vs), h(vz), ko, vo, n_rows, seqlen,
                                                 kv_buf_len, gs, n_groups_buf, vec);
    else if (fmt == 1)
        dequant_kernel<1><<<nb, 256, 0, stream>>>(c(kq), h(ks), h(kz), c(vq), h(vs), h(vz), ko, vo, n_rows, seqlen,
                                                 kv_buf_len, gs, n_groups_buf, vec);
    else
        dequant_kernel<2><<<nb, 256, 0, stream>>>(c(kq), h(ks), h(kz), c(vq), h(vs), h(vz), ko, vo, n_rows, seqlen,
                                                 kv_buf_len, gs, n_groups_buf, vec);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        err = std::string("dequantize launch: ") + cudaGetErrorString(e);
        return LIK_ERR_CUDA;
    }
    return LIK_OK;
}

}  // namespace lik
