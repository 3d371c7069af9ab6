// Rotary positions of query and key heads, both in one launch:
//   (x_a, x_b) -> gain * (x_a cos t - x_b sin t, x_b cos t + x_a sin t),   t = position * inv_freq[pair]
// for the pairs of a head's first 2 n columns -- (i, i + n) in the half layout, (2i, 2i + 1) in the interleaved one; the other columns are
// copied.  With two positions per token (row and column of an image token) the first half of the pairs turns by the first, the rest by the
// second.  The gradient is the same turn by -t.
// Bound by HBM: every element is read and written once.  The angle is reduced in 64 bits (t / 2 pi minus the nearest whole number: at
// position 10^6 a product in 32 bits is off by 0.03 rad) and the sine and cosine are taken of the remainder, once per token and pair for
// all heads: a workgroup puts the table of its tokens in LDS, then streams the heads, eight pairs (two 16-byte vectors of 16-bit
// data) per thread and step.  16384 tokens x 40 heads of 128, bf16: 71 to 79 us, 4.7 to 4.2 TB/s.
#include "token_types.hpp"

using namespace casmtr;

namespace {
struct RotArgs {
    const void *q, *k, *pos;
    void *oq, *ok;
    const double* freq;
    long long T, q_ts, q_hs, k_ts, k_hs;   // token and head strides, in elements
    int Hq, Hk, D, n, axes, pos64, layout, tpw;
    float gain, sign;
};

constexpr int ROT_TABLE = 1024;   // (token, pair) entries of a workgroup's table

template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs a) {
    __shared__ float s_cos[ROT_TABLE], s_sin[ROT_TABLE];
    const long long t0 = (long long)blockIdx.x * a.tpw;
    const int nt = (int)min((long long)a.tpw, a.T - t0);
    for (int i = threadIdx.x; i < nt * a.n; i += 256) {
        const int tok = i / a.n, p = i - tok * a.n;
        const long long pi = (t0 + tok) * a.axes + (a.axes == 2 && p >= a.n / 2 ? 1 : 0);
        const double pos = a.pos64 ? (double)((const long long*)a.pos)[pi] : (double)((const int*)a.pos)[pi];
        const double turns = pos * a.freq[p] * 0.15915494309189533577;
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        s_cos[i] = cs * a.gain;
        s_sin[i] = sn * a.gain * a.sign;
    }
    __syncthreads();
    const int ni = (a.n + 7) / 8, nc = (a.D - 2 * a.n + 15) / 16, per = ni + nc, heads = a.Hq + a.Hk;
    for (int it = threadIdx.x; it < nt * heads * per; it += 256) {
        const int hd = it / per, c = it - hd * per, tok = hd / heads, h = hd - tok * heads;
        const long long t = t0 + tok;
        const T* src = h < a.Hq ? (const T*)a.q + t * a.q_ts + h * a.q_hs : (const T*)a.k + t * a.k_ts + (h - a.Hq) * a.k_hs;
        T* dst = h < a.Hq ? (T*)a.oq + (t * a.Hq + h) * a.D : (T*)a.ok + (t * a.Hk + h - a.Hq) * a.D;
        float u[8], v[8];
        if (c >= ni) {   // columns that do not rotate
            const int col = 2 * a.n + 16 * (c - ni), m = a.D - col;
            load_n(src + col, u, m);
            if (m > 8) load_n(src + col + 8, v, m - 8);
            store_n(dst + col, u, m);
            if (m > 8) store_n(dst + col + 8, v, m - 8);
            continue;
        }
        const int p = 8 * c, m = min(8, a.n - p);
        const float *cs = s_cos + tok * a.n + p, *sn = s_sin + tok * a.n + p;
        if (a.layout == CASMTR_ROTARY_HALF) {
            load_n(src + p, u, m);
            load_n(src + a.n + p, v, m);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int f = e < m ? e : 0;
                const float x = u[e], y = v[e];
                u[e] = x * cs[f] - y * sn[f];
                v[e] = y * cs[f] + x * sn[f];
            }
            store_n(dst + p, u, m);
            store_n(dst + a.n + p, v, m);
        } else {
            load_n(src + 2 * p, u, 2 * m);
            if (m > 4) load_n(src + 2 * p + 8, v, 2 * m - 8);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int f = e < m ? e : 0, g = e + 4 < m ? e + 4 : 0;
                float x = u[2 * e], y = u[2 * e + 1];
                u[2 * e] = x * cs[f] - y * sn[f];
                u[2 * e + 1] = y * cs[f] + x * sn[f];
                x = v[2 * e], y = v[2 * e + 1];
                v[2 * e] = x * cs[g] - y * sn[g];
                v[2 * e + 1] = y * cs[g] + x * sn[g];
            }
            store_n(dst + 2 * p, u, 2 * m);
            if (m > 4) store_n(dst + 2 * p + 8, v, 2 * m - 8);
        }
    }
}
}  // namespace

extern "C" int casmtr_rotary_fwd(const void* q, const void* k, const void* pos, const double* inv_freq, void* oq, void* ok, long long T, int Hq, int Hk,
                                 int D, int npairs, int axes, int pos_is_i64, int layout, float gain, int inverse, long long q_token_stride,
                                 long long q_head_stride, long long k_token_stride, long long k_head_stride, int dtype, casmtr_stream_t stream) {
    if (T < 0 || Hq < 0 || Hk < 0 || D <= 0 || npairs <= 0 || 2 * (long long)npairs > D || npairs > ROT_TABLE || (axes != 1 && axes != 2) ||
        (axes == 2 && npairs % 2 != 0) || (layout != CASMTR_ROTARY_HALF && layout != CASMTR_ROTARY_INTERLEAVED) ||
        ((long long)Hq + Hk) * D > (1LL << 24))
        return CASMTR_ERR_UNSUPPORTED;
    if (T == 0 || Hq + Hk == 0) return 0;
    // tokens per workgroup: two, more where that leaves the threads without four steps each, as many as the table holds, fewer where the CUs would
    // not get a few workgroups each (16384 tokens x 40 heads of 128, 64 columns interleaved, bf16, 1 / 2 / 4 / 8 / 16 tokens: 74 / 71 / 74 / 75 / 83 us)
    const int steps = (Hq + Hk) * ((npairs + 7) / 8 + (D - 2 * npairs + 15) / 16);   // of a token
    int tpw = 1024 / steps > 2 ? 1024 / steps : 2;
    if (tpw > ROT_TABLE / npairs) tpw = ROT_TABLE / npairs;
    while (tpw > 1 && T / tpw < 1024) tpw >>= 1;
    const long long wgs = (T + tpw - 1) / tpw;
    if (wgs > 0x7fffffffLL) return CASMTR_ERR_UNSUPPORTED;
    RotArgs a{q, k, pos, oq, ok, inv_freq, T, q_token_stride, q_head_stride, k_token_stride, k_head_stride, Hq, Hk, D, npairs, axes, pos_is_i64, layout, tpw,
              gain, inverse ? -1.f : 1.f};
    ProfScope ps(CASMTR_PROF_GLUE, (hipStream_t)stream, "rotary_kernel");
    if (!with_type(dtype, [&](auto tv) {
            hipLaunchKernelGGL((rotary_kernel<decltype(tv)>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, a);
        }))
        return CASMTR_ERR_UNSUPPORTED;
    CASMTR_CHECK_LAUNCH();
    return 0;
}
