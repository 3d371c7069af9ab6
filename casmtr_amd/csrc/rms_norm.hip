// Root-mean-square norm over the last axis, with the residual's addition in front and, on request, an 8-bit output with scales behind it;
// and its gradient.
//   h = round(x + r);  y = h * rstd * w,  rstd = 1 / sqrt(mean(h^2) + eps);  scale = max|y| / top (per row or per block of columns),
//   q = round8(y / scale).
//   dx = (g - n * mean(g n)) * rstd + dh,  g = dy w,  n = h rstd;   dw = sum over rows of dy n.
// Bound by HBM: a row is read once, kept in registers (CH chunks of 8 elements per thread) between the sum of squares and the output,
// and everything a row needs is one launch.  A row belongs to one wave up to 1024 columns (the reduction is 6 DPP steps, no barrier),
// to a workgroup of 256 threads up to 8192, of 1024 threads up to 16384 (with 256 the gradient's kernel needs 284 registers per thread).
// 8192 x 4096 bf16 with residual 50 us (41 to 52, 5.4 TB/s); 16384 x 8192 into e4m3 with scales for 128 columns 179 us (5.2 TB/s).
// Sums are fp32 in a fixed order; the weight's gradient is reduced without atomics (per-workgroup partial sums in the workspace, then one
// column-wise pass), so results repeat bit for bit.
#include "token_types.hpp"

using namespace casmtr;

namespace {

struct NormArgs {
    const void *x, *res, *w;
    void *y, *h;
    float *rstd, *scale;
    long long rows, xs, rs;   // row strides of x and res, in elements
    int C, w_f32, quant, group;
    float eps, inv_c;
};

__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
    v = max(v, wave_xor_u32<1>(v)); v = max(v, wave_xor_u32<2>(v)); v = max(v, wave_xor_u32<4>(v));
    v = max(v, wave_xor_u32<8>(v)); v = max(v, wave_xor_u32<16>(v)); v = max(v, wave_xor_u32<32>(v));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
    v += __uint_as_float(wave_xor_u32<1>(__float_as_uint(v))); v += __uint_as_float(wave_xor_u32<2>(__float_as_uint(v)));
    v += __uint_as_float(wave_xor_u32<4>(__float_as_uint(v))); v += __uint_as_float(wave_xor_u32<8>(__float_as_uint(v)));
    v += __uint_as_float(wave_xor_u32<16>(__float_as_uint(v))); v += __uint_as_float(wave_xor_u32<32>(__float_as_uint(v)));
    return v;
}
// sum / max over the TPR threads of a row; `slot` is an LDS array of TPR / 64 words that nothing else uses between two barriers
template <int TPR>
__device__ __forceinline__ float row_add(float v, float* slot) {
    v = wave_add(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += slot[i];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ unsigned row_max(unsigned v, unsigned* slot) {
    v = wave_max_u32(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v = max(v, slot[i]);
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void load_w(const void* w, int w_f32, int col, int n, float (&v)[8]) {
    if (w_f32) load_n((const float*)w + col, v, n);
    else load_n((const T*)w + col, v, n);
}

// eight values to 8 bits: out of range goes to the largest value (a division by the scale can round up past it), NaN stays
__device__ __forceinline__ void store_q8(unsigned char* p, const float (&v)[8], int n, int quant) {
    const float top = quant == CASMTR_Q_E4M3 ? 448.f : quant == CASMTR_Q_E5M2 ? 57344.f : 127.f;
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = v[i] > top ? top : (v[i] < -top ? -top : v[i]);
    unsigned char b[8];
    if (quant == CASMTR_Q_I8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (unsigned char)(signed char)(int)rintf(c[i]);
    } else {
        int lo = 0, hi = 0;
        if (quant == CASMTR_Q_E4M3) {
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], lo, false); lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], hi, false); hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
        } else {
            lo = __builtin_amdgcn_cvt_pk_bf8_f32(c[0], c[1], lo, false); lo = __builtin_amdgcn_cvt_pk_bf8_f32(c[2], c[3], lo, true);
            hi = __builtin_amdgcn_cvt_pk_bf8_f32(c[4], c[5], hi, false); hi = __builtin_amdgcn_cvt_pk_bf8_f32(c[6], c[7], hi, true);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { b[i] = (unsigned char)(lo >> (8 * i)); b[4 + i] = (unsigned char)(hi >> (8 * i)); }
    }
    if (n >= 8) {
        typedef unsigned char u8x8 __attribute__((ext_vector_type(8), aligned(1)));
        u8x8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = b[i];
        *reinterpret_cast<u8x8*>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = b[i];
    }
}

__device__ __forceinline__ float q8_scale(unsigned amax_bits, int quant) {
    const float top = quant == CASMTR_Q_E4M3 ? 448.f : quant == CASMTR_Q_E5M2 ? 57344.f : 127.f;
    const float s = __fdiv_rn(__uint_as_float(amax_bits), top);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;   // a row of zeros: the smallest normal number, whose reciprocal is finite (NaN stays)
}

// y / scale, correctly rounded but for quotients within 2^-46 of a border between two: the product with the reciprocal, which next to a border between
// two codes is on the wrong side now and then, and one step with its remainder.  (16384 x 8192 into e4m3 with scales for 128 columns, call by call: the
// division's own instructions 207 us, this 195, the product alone 191.)
struct Quotient {
    float sc, inv;   // sc: 0 for an infinite scale, which leaves the product (0, or NaN of an infinity) as it is
    __device__ __forceinline__ explicit Quotient(float scale) : sc(scale < INFINITY ? scale : 0.f), inv(1.0f / scale) {}
    __device__ __forceinline__ float operator()(float y) const {
        const float q = y * inv;
        return __builtin_fmaf(__builtin_fmaf(-q, sc, y), inv, q);
    }
};

// TPR threads per row, CH chunks of 8 columns per thread: chunk i of thread t covers columns 8 (t + TPR i) .. + 7
template <typename T, int TPR, int CH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(const NormArgs a) {
    constexpr int RPW = TPR < 256 ? 256 / TPR : 1;
    __shared__ float s_sum[TPR < 256 ? 1 : TPR / 64];
    __shared__ unsigned s_max[TPR < 256 ? 1 : TPR / 64];
    __shared__ float s_big[TPR < 256 ? 1 : TPR / 64];
    const int t = threadIdx.x % TPR;
    const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RPW + threadIdx.x / TPR;
    if (row >= a.rows) return;   // whole waves only where a row is a wave's, the whole workgroup never otherwise
    const T* xr = (const T*)a.x + row * a.xs;
    const T* rr = a.res ? (const T*)a.res + row * a.rs : nullptr;
    float v[CH][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int col = 8 * (t + TPR * i), n = a.C - col;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        if (n > 0) {
            load_n(xr + col, v[i], n);
            if (rr) {
                float r[8];
                load_n(rr + col, r, n);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = (float)(T)(v[i][e] + r[e]);   // the stream is handed on in its own type; the norm is of what is handed on
                store_n((T*)a.h + row * a.C + col, v[i], n);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(v[i][e], v[i][e], s);
    }
    s = row_add<TPR>(s, s_sum);
    float rstd = 1.0f / sqrtf(s * a.inv_c + a.eps);
    if (!(s < INFINITY)) {   // (the same for the whole row) squares past fp32, from |h| = 1.8e19 on: of 2^-80 h, beside which eps is nothing
        s = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(v[i][e] * 0x1p-80f, v[i][e] * 0x1p-80f, s);
        rstd = 0x1p-80f / sqrtf(row_add<TPR>(s, s_big) * a.inv_c);
    }
    if (a.rstd && t == 0) a.rstd[row] = rstd;
    unsigned big = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int col = 8 * (t + TPR * i), n = a.C - col;
        if (n > 0) {
            float w[8];
            load_w<T>(a.w, a.w_f32, col, n, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * rstd * w[e];
        }
        if (!a.quant) {
            if (n > 0) store_n((T*)a.y + row * a.C + col, v[i], n);
            continue;
        }
        unsigned m = 0;   // max |y| as bits: NaN is above infinity, so it reaches the scale
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[i][e]) & 0x7fffffffu);
        if (a.group) {    // 128 columns = the 16 chunks of one 16-lane row of the wave
            m = max(m, dpp_u32<0xB1>(m)); m = max(m, dpp_u32<0x4E>(m)); m = max(m, dpp_u32<0x141>(m)); m = max(m, dpp_u32<0x140>(m));
            const float sc = q8_scale(m, a.quant);
            if (n > 0) {
                if ((t & 15) == 0) a.scale[row * (a.C / 128) + col / 128] = sc;
                const Quotient by(sc);
                float q[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e] = by(v[i][e]);
                store_q8((unsigned char*)a.y + row * a.C + col, q, n, a.quant);
            }
        } else big = max(big, m);
    }
    if (!a.quant || a.group) return;
    const float sc = q8_scale(row_max<TPR>(big, s_max), a.quant);
    const Quotient by(sc);
    if (t == 0) a.scale[row] = sc;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int col = 8 * (t + TPR * i), n = a.C - col;
        if (n <= 0) continue;
        float q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = by(v[i][e]);
        store_q8((unsigned char*)a.y + row * a.C + col, q, n, a.quant);
    }
}

struct NormBwdArgs {
    const void *dy, *dh, *h, *w;
    const float* rstd;
    void* dx;
    float* part;              // [parts, C] partial sums of dw
    long long rows, dys, dhs, hs;
    int C, w_f32;
    float inv_c;
};

// Part p (a workgroup; a wave where TPR == 64) takes the rows p, p + parts, ... and keeps its share of dw in registers.
template <typename T, int TPR, int CH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int RPW = TPR < 256 ? 256 / TPR : 1;
    __shared__ float s_sum[2][TPR < 256 ? 1 : TPR / 64];
    const int t = threadIdx.x % TPR;
    const long long part = (long long)blockIdx.x * RPW + threadIdx.x / TPR, parts = (long long)gridDim.x * RPW;
    float dw[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
    int turn = 0;
    for (long long row = part; row < a.rows; row += parts, turn ^= 1) {
        const float rstd = a.rstd[row];
        float g[CH][8], nn[CH][8], c = 0.f;
        vec8_t<T> dh[CH];   // loaded with the rest, before the row's sum is waited for
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int col = 8 * (t + TPR * i), n = a.C - col;
            if (n > 0) {
                load_n((const T*)a.dy + row * a.dys + col, g[i], n);
                load_n((const T*)a.h + row * a.hs + col, nn[i], n);
                if (a.dh) dh[i] = load_raw_n((const T*)a.dh + row * a.dhs + col, n);
            }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int col = 8 * (t + TPR * i), n = a.C - col;
            if (n > 0) {
                float w[8];
                load_w<T>(a.w, a.w_f32, col, n, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    nn[i][e] *= rstd;
                    dw[i][e] = fmaf(g[i][e], nn[i][e], dw[i][e]);
                    g[i][e] *= w[e];
                    c = fmaf(g[i][e], nn[i][e], c);
                }
            }
        }
        c = row_add<TPR>(c, s_sum[turn]) * a.inv_c;   // two slots in turn: a row's sum is read behind ONE barrier
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int col = 8 * (t + TPR * i), n = a.C - col;
            if (n <= 0) continue;
            float d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = a.dh ? (float)dh[i][e] : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(g[i][e] - nn[i][e] * c, rstd, d[e]);
            store_n((T*)a.dx + row * a.C + col, d, n);
        }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int col = 8 * (t + TPR * i), n = a.C - col;
        if (n > 0) store_n(a.part + part * a.C + col, dw[i], n);
    }
}

// dw[c] = sum of the partial sums' column c: 32 columns x 32 row lanes per workgroup, lanes joined in LDS in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* __restrict__ part, T* __restrict__ dw, int parts, int C) {
    __shared__ float s[32][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
    float acc = 0.f;
    if (c < C)
        for (int p = ry; p < parts; p += 32) acc += part[(long long)p * C + c];
    s[ry][cx] = acc;
    __syncthreads();
    if (ry == 0 && c < C) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) v += s[i][cx];
        dw[c] = (T)v;
    }
}

// f(TPR, CH) as compile-time constants for a row of C columns; -> false beyond 16384
template <typename F>
bool with_row_shape(int C, F&& f) {
    const int c8 = (C + 7) / 8;
    using std::integral_constant;
    if (c8 <= 64) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (c8 <= 128) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (c8 <= 256) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (c8 <= 512) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (c8 <= 1024) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else if (c8 <= 2048) f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    else return false;
    return true;
}

// parts of the weight's gradient: one per workgroup (wave), as many as keep the chip full and no more than there are rows (8192 x 4096 bf16 with dh,
// both kernels, at most 256 / 512 / 768 / 1024 / 2048 workgroups: 139 / 87 / 77 / 71 / 81 us, 4.8 TB/s at 1024)
int bwd_parts(long long rows, int C) {
    const int rpw = (C + 7) / 8 <= 128 ? 4 : 1;
    long long wgs = (rows + rpw - 1) / rpw;
    if (wgs > 1024) wgs = 1024;
    return (int)(wgs * rpw);
}
}  // namespace

extern "C" int casmtr_rms_norm_fwd(const void* x, const void* residual, const void* w, void* y, void* h, float* rstd, float* scale,
                                   long long rows, int C, long long x_stride, long long r_stride, float eps, int dtype, int w_dtype, int quant,
                                   int group, casmtr_stream_t stream) {
    if (rows < 0 || rows > 0x7fffffffLL || C <= 0 || quant < 0 || quant > CASMTR_Q_I8 || (group != 0 && (group != 128 || C % 128 != 0 || !quant)) ||
        (w_dtype != CASMTR_F32 && w_dtype != dtype))
        return CASMTR_ERR_UNSUPPORTED;
    if (rows == 0) return 0;   // (no rows, no pointers)
    if ((quant && !scale) || (residual && !h)) return CASMTR_ERR_UNSUPPORTED;
    NormArgs a{x, residual, w, y, h, rstd, scale, rows, x_stride, r_stride, C, w_dtype == CASMTR_F32, quant, group, eps, 1.0f / (float)C};
    bool ok = false;
    ProfScope ps(CASMTR_PROF_GLUE, (hipStream_t)stream, "rms_norm_kernel");
    if (!with_type(dtype, [&](auto tv) {
            typedef decltype(tv) T;
            ok = with_row_shape(C, [&](auto tpr, auto ch) {
                constexpr int TPR = decltype(tpr)::value, CH = decltype(ch)::value, RPW = TPR < 256 ? 256 / TPR : 1;
                const long long wgs = (rows + RPW - 1) / RPW, x = wgs < (1 << 21) ? wgs : 1 << 21;   // (a launch's x holds 2^32 threads)
                hipLaunchKernelGGL((rms_norm_kernel<T, TPR, CH>), dim3((unsigned)x, (unsigned)((wgs + x - 1) / x)), dim3(TPR < 256 ? 256 : TPR), 0,
                                   (hipStream_t)stream, a);
            });
        }) || !ok)
        return CASMTR_ERR_UNSUPPORTED;
    CASMTR_CHECK_LAUNCH();
    return 0;
}

extern "C" size_t casmtr_rms_norm_bwd_ws_floats(long long rows, int C) { return rows <= 0 || C <= 0 ? 0 : (size_t)bwd_parts(rows, C) * C; }

extern "C" int casmtr_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* rstd, void* dx, void* dw, float* ws,
                                   long long rows, int C, long long dy_stride, long long dh_stride, long long h_stride, int dtype, int w_dtype,
                                   casmtr_stream_t stream) {
    if (rows <= 0 || C <= 0 || rows > 0x7fffffffLL || !rstd || !ws || (w_dtype != CASMTR_F32 && w_dtype != dtype)) return CASMTR_ERR_UNSUPPORTED;
    NormBwdArgs a{dy, dh, h, w, rstd, dx, ws, rows, dy_stride, dh_stride, h_stride, C, w_dtype == CASMTR_F32, 1.0f / (float)C};
    const int parts = bwd_parts(rows, C);
    bool ok = false;
    ProfScope ps(CASMTR_PROF_GLUE, (hipStream_t)stream, "rms_norm_bwd_kernel, rms_norm_dw_kernel");
    if (!with_type(dtype, [&](auto tv) {
            typedef decltype(tv) T;
            ok = with_row_shape(C, [&](auto tpr, auto ch) {
                constexpr int TPR = decltype(tpr)::value, CH = decltype(ch)::value, RPW = TPR < 256 ? 256 / TPR : 1;
                hipLaunchKernelGGL((rms_norm_bwd_kernel<T, TPR, CH>), dim3(parts / RPW), dim3(TPR < 256 ? 256 : TPR), 0, (hipStream_t)stream, a);
            });
        }) || !ok)
        return CASMTR_ERR_UNSUPPORTED;
    CASMTR_CHECK_LAUNCH();
    with_type(w_dtype, [&](auto tv) {
        typedef decltype(tv) T;
        hipLaunchKernelGGL((rms_norm_dw_kernel<T>), dim3((C + 31) / 32), dim3(1024), 0, (hipStream_t)stream, ws, (T*)dw, parts, C);
    });
    CASMTR_CHECK_LAUNCH();
    return 0;
}
