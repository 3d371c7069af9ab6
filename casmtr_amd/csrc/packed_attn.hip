// Attention over packed sequences of different lengths, forward:
//   o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j) over the keys j that row i sees,  lse_i = log sum_j exp(scale q_i . k_j)
// Row i of a sequence with nq rows and nk keys sees all keys, or, causal, the keys j <= i + nk - nq.  A row that sees none gives 0 and -inf.
// Query heads share key heads in groups of G = H / Hk.
//
// fp32 runs as three bf16 terms (x3_t) -- 8 x 43264 rows x 676 keys, 4 heads of 32: 0.76 ms in a row of calls, 0.83 in a kernel trace of five (158 and 145
// TFLOP/s) against 1.12 ms on the fp32 matrix instructions, whose 154 TFLOP/s bound it --, except for few rows, where the reads bound it.
//
// One pass over the keys with the running maximum and sum of the softmax.  A tile's rows are (token, head of the group) pairs, token-major, so
// all G heads of a key head use one copy of its keys, and a single token of G heads is one tile.  A workgroup has four waves of 32 rows; K and V
// tiles of BN keys go through LDS in two stages: the next tile's loads are in flight while this one is multiplied, one barrier per tile.
// Bound by the matrix instructions (heads of 128: 53 % of the cycles are theirs at the clock that they leave, 1.8 GHz) and, for smaller heads, by the
// exponentials: 32 of 16 cycles each beside 512 cycles of matrix instructions per tile of 64 keys and wave at 64 columns.  So registers are kept
// to two (64 and less: three) waves per SIMD that take turns; with two, heads of 64 ran at 752 in place of 860 TFLOP/s.  16384 causal tokens,
// 32 / 8 heads of 128: bf16 2.16 ms (1.02 PFLOP/s), fp16 2.21 (0.99; a library product of 8192^3: 1.05), the first calls on a cold card up to 2.45.
// LDS conflicts: none.
#include "packed_attn.hpp"

using namespace casmtr;

namespace {
struct AttnArgs {
    const void *q, *k, *v;
    void* o;
    float* lse;                        // [Tq, H] or NULL
    float *part_o, *part_ml;           // splits > 1: [splits, Tq * H, D] and [splits, Tq * H, 2]
    PackedSeqs s;
    long long qts, qhs, kts, khs, vts, vhs;   // token and head strides, in elements
    int H, Hk, D, splits;
    float scale;                       // times log2(e): scores are in bits
};

constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;
constexpr float RESCALE_AT = 8.f;   // the accumulator is rescaled only when a maximum grew by more than 8 bits: exp2 stays below 256, far from any overflow
// Probabilities are multiplied as 2^P_BITS of their value: in fp16 they stay in the normal range down to 2^-21 of the row's largest then, and what is lost
// below that is at most 2^-32 of it each -- beside 2^-25 without, which 65536 keys of 2^-25 make up to a whole result.  2^(RESCALE_AT + 7) is within
// fp16.  The row's sum carries the same factor, so only lse has to take it out.
template <typename T> constexpr float P_BITS = std::is_same<T, f16_t>::value ? 7.f : 0.f;

// FEW (few rows, long keys): a workgroup has 32 rows, its waves take 32 keys each of a tile and are joined in LDS at the end.  With 128 rows per
// workgroup a tile takes each wave the whole way through 64 keys, for nothing where three of four waves have no rows of their own.
template <typename T, int DP, int BN, int NW, bool DMA, bool FEW>
__global__ __launch_bounds__(64 * NW, !FEW && (sizeof(T) == 2 || (sizeof(T) == 1 && DP <= 64)) ? (sizeof(T) == 2 && DP <= 64 ? 3 : 2) : 1) void packed_attn_kernel(const AttnArgs a) {
    typedef Tile<T, DP, BN> L;
    static_assert(!FEW || BN == 32 * NW, "one block of keys per wave");
    constexpr int BM = FEW ? 32 : 32 * NW, KS = DP / 16, NB = FEW ? 1 : BN / 32, DB = DP / 32;
    __shared__ __attribute__((aligned(256))) char smem[TilePair<T, DP, BN, NW, DMA>::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, r = lane & 31;
    const int hk = blockIdx.x % a.Hk, G = a.s.G;
    int tile;
    const int seq = seq_of_slot(a.s.cu_q, a.s.n, a.s.Tq, G, BM, (long long)(gridDim.x / a.Hk - 1 - blockIdx.x / a.Hk), &tile);   // later rows see more keys: first
    const Span rows = span_of(a.s.cu_q, seq, a.s.n, a.s.Tq), keys = keys_of(a.s, seq);
    const int nrow = rows.count * G;
    if ((long long)tile * BM >= nrow) return;   // a slot too many
    const int row0 = tile * BM;
    const int wrow = FEW ? 0 : 32 * wave, wkey = FEW ? 32 * wave : 0;   // the wave's rows of the workgroup's, keys of a tile's
    const int row = row0 + wrow + r, rc = min(row, nrow - 1), tok = rc / G, head = hk * G + rc % G;
    const int shift = keys.count - rows.count;
    const int limit = a.s.causal ? max(0, min(keys.count, tok + shift + 1)) : keys.count;   // this lane's row sees the keys [0, limit)
    // keys that some row of the workgroup / of the wave sees (rows see more the later they are), keys that all rows of the wave see
    const auto limit_at = [&](int rr) { return a.s.causal ? max(0, min(keys.count, min(rr, nrow - 1) / G + shift + 1)) : keys.count; };
    const int wg_end = limit_at(row0 + BM - 1), wave_end = limit_at(row0 + wrow + 31), wave_all = limit_at(row0 + wrow);
    int t0 = 0, t1 = (wg_end + BN - 1) / BN;
    if (a.splits > 1) {
        const int per = (t1 + a.splits - 1) / a.splits;
        t0 = min(t1, per * (int)blockIdx.y);
        t1 = min(t1, t0 + per);
    }
    TilePair<T, DP, BN, NW, DMA> kv;
    kv.init(smem, tid, wave, a.kts, a.vts, a.D);
    kv.of((const store_t<T>*)a.k + (long long)keys.begin * a.kts + hk * a.khs, (const store_t<T>*)a.v + (long long)keys.begin * a.vts + hk * a.vhs, keys.count);
    if (t0 < t1) kv.fetch(t0, 0);
    frag_t<T> qf[KS];
    const auto load_q = [&](auto guard) {
        const store_t<T>* qr = (const store_t<T>*)a.q + (long long)(rows.begin + tok) * a.qts + head * a.qhs;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_frag<T, decltype(guard)::value>(qr, s, h, a.D);
    };
    load_q(std::false_type{});
    f32x16 acc[DB];
    float m, l;
    // One pass over the keys.  GUARD: with the product that keeps what a row does not see away from it (mma_hidden)
    const auto pass = [&](auto guard) {
        constexpr bool GUARD = decltype(guard)::value;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = zero16();
        m = -INFINITY;
        l = 0.f;
        if (GUARD && std::is_same<T, x3_t>::value) load_q(guard);
        if (GUARD && t0 < t1) kv.fetch(t0, 0);   // (the first pass's first tile is under way)
        const auto step = [&](int t, auto stage_) {
            constexpr int stage = decltype(stage_)::value;   // a constant: it goes into the offsets of the LDS reads
            kv.template arrived<GUARD>(stage);
            __syncthreads();   // this tile is in LDS; nobody reads the other stage any more
            if (t + 1 < t1) kv.fetch(t + 1, stage ^ 1);
            const int key0 = t * BN + wkey;
            if (key0 >= wave_end) return;
            const bool hidden = key0 + 32 * NB > wave_all;   // some pair of the wave's is hidden
            {
                const char *ks = kv.first(stage), *vs = kv.second(stage);
                f32x16 s[NB];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    s[b] = zero16();
#pragma unroll
                    for (int st = 0; st < KS; ++st) {
                        const frag_t<T> kf = L::rows(ks, wkey + 32 * b + r, st, h);
                        s[b] = GUARD ? mma_any<T>(kf, qf[st], s[b], h) : mma(kf, qf[st], s[b]);
                    }
                }
                if (hidden) {
                    const int lim = limit - key0 - 4 * h;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[b][i] = seen_or(s[b][i], -INFINITY, 32 * b + 8 * (i >> 2) + (i & 3), lim);
                }
                float big[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = b ? 0 : 4; i < 16; ++i) big[i & 3] = fmaxf(big[i & 3], s[b][i]);
                const float mx = max_halves(fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]))) * a.scale;
                const bool up = mx > m + RESCALE_AT;   // (also the first tile: m = -inf); per row, so that a row's bits do not depend on its neighbours
                if (__any(up)) {
                    const float f = !up ? 1.f : m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
                    m = up ? mx : m;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[d][i] *= f;
                }
                const float mm = m == -INFINITY ? 0.f : m - P_BITS<T>;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};   // four chains: one would wait for every addition
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], a.scale, -mm));
                        sum[i & 3] += s[b][i];
                    }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
                        const frag_t<T> p = to_frag<T>(s[b], tt);   // probabilities below 256 (2^15 with P_BITS) rounded to the values' type; l sums the unrounded ones
                        const int k0 = 32 * b + 16 * tt;
#pragma unroll
                        for (int d = 0; d < DB; ++d) {
                            const frag_t<T> vt = L::cols(vs, wkey + k0, 32 * d, lane);
                            if constexpr (!GUARD) acc[d] = mma(vt, p, acc[d]);
                            else acc[d] = mma_hidden<T>(vt, p, acc[d], h, [&](int n) { return key0 + k0 + 8 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3) < limit; });
                        }
                    }
            }
        };
        for (int t = t0; t < t1; t += 2) {
            step(t, std::integral_constant<int, 0>{});
            if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
        }
    };
    pass(std::false_type{});
    // Hidden keys are weighted with exact zeros, so an infinity or NaN among hidden values is the only way by which one can reach a row that
    // does not see it -- and then the row's sum is not finite.  Rare enough to do it again, carefully, when that is seen.
    if (a.s.causal || std::is_same<T, x3_t>::value) {   // (three terms turn an infinity into NaN: that is done again too)
        float worst = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) worst += __builtin_fabsf(acc[d][i]);
        if (__syncthreads_or(!(worst < INFINITY))) pass(std::true_type{});
    }
    l = add_halves(l);
    if constexpr (FEW) {
        // join the waves: a row's maximum over them, every wave's share times 2^(m - maximum), the shares added in order
        constexpr int LD = DP + 4;
        static_assert((NW * 32 * LD + 2 * NW * 32) * 4 <= TilePair<T, DP, BN, NW, DMA>::BYTES, "the shares fit the tiles' LDS");
        float *share = reinterpret_cast<float*>(smem), *stat = share + NW * 32 * LD;
        __syncthreads();
        if (h == 0) { stat[wave * 32 + r] = m; stat[(NW + wave) * 32 + r] = l; }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(share + (wave * 32 + r) * LD + 32 * d + 8 * g + 4 * h) =
                    f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
        __syncthreads();
        constexpr int CT = DP / 4;   // threads of a row: four columns each
        for (int i = tid; i < 32 * CT; i += 64 * NW) {
            const int rr = i / CT, c = 4 * (i % CT);
            if (row0 + rr >= nrow) continue;
            float M = -INFINITY, w[NW], ls = 0.f;
#pragma unroll
            for (int j = 0; j < NW; ++j) M = fmaxf(M, stat[j * 32 + rr]);
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                const float mj = stat[j * 32 + rr], lj = stat[(NW + j) * 32 + rr];
                // m of -inf: the wave saw no key (its sums are zeros) or none of weight.  A share is added whatever its weight: where that underflows, an
                // infinity or NaN in it still reaches the row, as it does where one wave walks all keys (0 * inf)
                w[j] = mj == -INFINITY ? (lj != lj ? lj : 0.f) : __builtin_amdgcn_exp2f(mj - M);
                const f32x4 x = *reinterpret_cast<const f32x4*>(share + (j * 32 + rr) * LD + c);
                ls += w[j] * lj;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += w[j] * x[e];
            }
            const long long at = (long long)(rows.begin + (row0 + rr) / G) * a.H + hk * G + (row0 + rr) % G;
            if (a.splits > 1) {
                float* po = a.part_o + ((long long)blockIdx.y * a.s.Tq * a.H + at) * a.D;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.D) po[c + e] = o[e];
                if (c == 0) {
                    float* ml = a.part_ml + 2 * ((long long)blockIdx.y * a.s.Tq * a.H + at);
                    ml[0] = M;
                    ml[1] = ls;
                }
                continue;
            }
            const bool some = ls > 0.f || ls != ls;
            const float inv = some ? 1.0f / ls : 0.f;
            store_t<T>* orow = (store_t<T>*)a.o + at * a.D;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.D) orow[c + e] = (store_t<T>)(o[e] * inv);
            if (a.lse && c == 0) a.lse[at] = some ? (M - P_BITS<T> + __builtin_amdgcn_logf(ls)) * LN2 : -INFINITY;
        }
        return;
    }
    if (row >= nrow) return;
    const long long out_row = (long long)(rows.begin + tok) * a.H + head;
    if (a.splits > 1) {
        float* po = a.part_o + ((long long)blockIdx.y * a.s.Tq * a.H + out_row) * a.D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * h;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.D) po[c + e] = acc[d][4 * g + e];
            }
        if (h == 0) {
            float* ml = a.part_ml + 2 * ((long long)blockIdx.y * a.s.Tq * a.H + out_row);
            ml[0] = m;
            ml[1] = l;
        }
        return;
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    store_t<T>* orow = (store_t<T>*)a.o + out_row * a.D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * h;
            typedef store_t<T> S;
            typedef S T4 __attribute__((ext_vector_type(4), aligned(sizeof(S))));
            T4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (S)(acc[d][4 * g + e] * inv);
            if (c + 4 <= a.D) *reinterpret_cast<T4*>(orow + c) = v;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.D) orow[c + e] = v[e];
        }
    if (a.lse && h == 0) a.lse[out_row] = l > 0.f || l != l ? (m - P_BITS<T> + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

// joins the splits of a row: weights 2^(m_s - max m); one wave per row, lane s holds the weight of split s (at most 64)
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_join_kernel(const AttnArgs a) {
    const long long rows = a.s.Tq * a.H, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    float ms = -INFINITY, ls = 0.f;
    if (lane < a.splits) {
        const float* ml = a.part_ml + 2 * (lane * rows + row);
        ms = ml[0];
        ls = ml[1];
    }
    const float m = wave_max_f32(ms);
    const float w = ms == -INFINITY ? (ls != ls ? ls : 0.f) : __builtin_amdgcn_exp2f(ms - m);
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    const float* po = a.part_o + row * a.D;
    for (int s = 0; s < a.splits; s += 4) {   // four splits' loads in flight
        float x0[4], x1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool on = s + j < a.splits;
            x0[j] = on && lane < a.D ? po[(s + j) * rows * a.D + lane] : 0.f;
            x1[j] = on && lane + 64 < a.D ? po[(s + j) * rows * a.D + lane + 64] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(w), min(s + j, 63)));
            const float lj = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(ls), min(s + j, 63)));
            if (s + j >= a.splits) continue;   // (weights of 0 are added too: see the join of the waves above)
            l += f * lj;
            o0 += f * x0[j];
            o1 += f * x1[j];
        }
    }
    const bool some = l > 0.f || l != l;
    const float inv = some ? 1.0f / l : 0.f;
    T* orow = (T*)a.o + row * a.D;
    if (lane < a.D) orow[lane] = (T)(o0 * inv);
    if (lane + 64 < a.D) orow[lane + 64] = (T)(o1 * inv);
    if (a.lse && lane == 0) a.lse[row] = some ? (m - P_BITS<T> + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

constexpr int FWD_NW = 4;

// Few rows: at most 32 (token, head of the group) rows per sequence on average.  With 256 keys or more per sequence the waves of a workgroup share the
// keys (FEW above); with fewer -- windows and the like, where neither four waves' rows nor four waves' keys are there -- a workgroup is one wave,
// for heads of up to 64 (wider ones: the ordinary kernel).  8192 windows of 25 tokens, 8 heads of 16, bf16: one wave 174 us, FEW with four 547,
// the ordinary kernel 435; 2048 x 32 rows x 128 keys, 8 heads of 128: 475, 637, 287.
bool few_rows(long long Tq, int n, int H, int Hk) { return Tq * (H / Hk) <= 32LL * n; }
bool long_keys(long long Tk, int n) { return Tk >= 256LL * n; }

// How many parts a sequence's keys are split into: enough workgroups to fill the chip when there are few rows, and several times that many for few
// rows, whose sequences may be of any length beside each other (16 single tokens against 161 to 32768 keys, 8 key heads of 128, bf16, up
// to 512 / 1024 / 2048 / 4096 workgroups: 274 / 275 / 253 / 259 us; against 32768 each: 369 / 371 / 379 / 389 us, 5.8 to 5.5 TB/s).  A part is no shorter than 256 keys on average, so that what it writes (a
// row of fp32 per query row) stays small beside what it reads.
int split_count(long long Tq, long long Tk, int n, int H, int Hk) {
    const bool few = few_rows(Tq, n, H, Hk) && long_keys(Tk, n);
    const long long bm = few ? 32 : 32 * FWD_NW, tiles = (Tq * (H / Hk) + bm - 1) / bm, wgs = (tiles > n ? tiles : n) * Hk;
    if (wgs >= 512 && !few) return 1;
    long long s = (few ? 2048 : 1024) / (wgs > 0 ? wgs : 1);
    const long long most = Tk / (n > 0 ? n : 1) / 256;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
}  // namespace

extern "C" size_t casmtr_packed_attn_ws_floats(long long Tq, long long Tk, int nseq, int H, int Hk, int D) {
    if (Tq <= 0 || Tk < 0 || nseq < 0 || H <= 0 || Hk <= 0 || D <= 0) return 0;
    const int s = split_count(Tq, Tk, nseq, H, Hk);
    return s > 1 ? (size_t)s * Tq * H * (D + 2) : 0;
}

extern "C" int casmtr_packed_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, float* ws, const int* cu_q, const int* cu_k,
                                      const int* len_k, long long Tq, long long Tk, int nseq, int H, int Hk, int D, long long qts, long long qhs,
                                      long long kts, long long khs, long long vts, long long vhs, float scale, int causal, int dtype,
                                      casmtr_stream_t stream) {
    if (Tq < 0 || Tk < 0 || nseq < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || D <= 0 || D > 128 || !(scale > 0.f) || !(scale * LOG2E < INFINITY) ||
        Tq > 0x7fffff00LL || Tk > 0x7fffff00LL || Tq * (H / Hk) > 0x7fffff00LL)
        return CASMTR_ERR_UNSUPPORTED;
    if (Tq == 0) return 0;
    const int splits = split_count(Tq, Tk, nseq, H, Hk), G = H / Hk;
    if (splits > 1 && !ws) return CASMTR_ERR_UNSUPPORTED;
    const bool few = few_rows(Tq, nseq, H, Hk) && long_keys(Tk, nseq), one = few_rows(Tq, nseq, H, Hk) && !few && D <= 64;
    const long long rows = Tq * H, wgs = slot_count(Tq, G, nseq, few || one ? 32 : 32 * FWD_NW) * Hk;
    if (wgs > 0x7fffffffLL) return CASMTR_ERR_UNSUPPORTED;
    AttnArgs a{q, k, v, o, lse, ws, ws ? ws + (long long)splits * rows * D : nullptr, {cu_q, cu_k, len_k, nseq, G, causal != 0, Tq, Tk},
               qts, qhs, kts, khs, vts, vhs, H, Hk, D, splits, scale * LOG2E};
    ProfScope ps(CASMTR_PROF_GLUE, (hipStream_t)stream, "packed_attn_kernel");
    const bool ok = with_type(dtype, [&](auto tv) {
        typedef decltype(tv) T;
        const dim3 grid((unsigned)wgs, (unsigned)splits);
        // LDS: at most 64 KB, two workgroups per CU (few rows of 128 columns in 16 bits with 128 KB, one workgroup: 379 -> 436 us as above);
        // fp32 heads of more than 64 (32 for few rows) columns take 64 to 128 KB
        typedef TileDma<T, 128, 128, FWD_NW> Dma;
        const bool dma = Dma::fits(k, kts, khs, D) && Dma::fits(v, vts, vhs, D);
#define FWD_LAUNCH(DP, BN, NW, FEW)                                                                                                  \
    do {                                                                                                                             \
        if (dma) hipLaunchKernelGGL((packed_attn_kernel<T, DP, BN, NW, true, FEW>), grid, dim3(64 * NW), 0, (hipStream_t)stream, a); \
        else hipLaunchKernelGGL((packed_attn_kernel<T, DP, BN, NW, false, FEW>), grid, dim3(64 * NW), 0, (hipStream_t)stream, a);    \
    } while (0)
        if (one) {
            if (D <= 32) FWD_LAUNCH(32, 32, 1, true);
            else FWD_LAUNCH(64, 32, 1, true);
        } else if (few) {
            if (D <= 32) FWD_LAUNCH(32, 128, 4, true);
            else if (D <= 64) FWD_LAUNCH(64, 128, 4, true);
            else FWD_LAUNCH(128, 64, 2, true);
        } else if constexpr (sizeof(T) == 2) {
            if (D <= 32) FWD_LAUNCH(32, 64, FWD_NW, false);
            else if (D <= 64) FWD_LAUNCH(64, 64, FWD_NW, false);
            else FWD_LAUNCH(128, 64, FWD_NW, false);
        } else {
            const dim3 block(64 * FWD_NW);
            if (D <= 32) hipLaunchKernelGGL((packed_attn_kernel<x3_t, 32, 64, FWD_NW, false, false>), grid, block, 0, (hipStream_t)stream, a);
            else if (D <= 64) hipLaunchKernelGGL((packed_attn_kernel<x3_t, 64, 32, FWD_NW, false, false>), grid, block, 0, (hipStream_t)stream, a);
            else hipLaunchKernelGGL((packed_attn_kernel<x3_t, 128, 32, FWD_NW, false, false>), grid, block, 0, (hipStream_t)stream, a);
        }
#undef FWD_LAUNCH
        if (splits > 1) hipLaunchKernelGGL((packed_attn_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    });
    if (!ok) return CASMTR_ERR_UNSUPPORTED;
    CASMTR_CHECK_LAUNCH();
    return 0;
}
