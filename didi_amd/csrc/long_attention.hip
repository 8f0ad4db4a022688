// Attention of any lengths: queries over keys / values of another length (an encoder's states), forward and backward, with right
// padding, key masks, a causal limit, keys shared by groups of heads, a learned relative position bias by buckets, and dropout.
//
//   visible(b, i, j) = j < count[b] and mask[b, j] != 0 and (not causal or j <= q_start + i)
//   t_ij  = scale q_i . k_j + table[bucket(j - q_start - i)][head]          p_ij = exp(t_ij - lse_i) over the visible j, 0 elsewhere
//   o_i   = sum_j drop(p_ij) v_j           lse_i = log sum_j exp(t_ij)
//   ds_ij = p_ij (drop(do_i . v_j) - do_i . o_i)
//   dq_i  = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i     dv_j = sum_i drop(p_ij) do_i     dtable[t][h] = sum of ds of bucket t
// A row that sees no key gives o = 0, lse = -inf and no gradients; keys and values that are not visible to a dialog are never
// multiplied (their LDS rows are zeros), so whatever lies there -- infinities, NaN -- stays there.
//
// One online softmax pass (running maximum and sum per row, fp32).  Everything is laid out so that one lane owns one row's statistics:
//   S^T = K Q^T   v_mfma_f32_32x32x16 (32x32x2 in fp32), A = K rows out of LDS, B = Q rows in registers
//                 -> lane holds t[q = lane & 31][key = (r & 3) + 8 (r >> 2) + 4 (lane >> 5)], r = 0..15
//   O^T += V^T P^T   the 16-bit probabilities a lane holds ARE its B operand (the contraction runs over the lane's own keys); the
//                 matching V^T operand comes out of the row-major V image by transposing LDS reads (fp32: plain row reads)
// so the rescale by exp(m_old - m_new) and every per-row constant of the backward is one register of the lane.
// The backward's dK / dV kernel is the mirror image (lane = key), its dQ kernel the forward's arrangement: two deterministic passes
// (14 products per pair and head-dim element against 10 with atomics, whose order would change the result).
#include <math.h>

#include <algorithm>
#include <mutex>

#include "common.hpp"
#include "philox.hpp"

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef short v4s __attribute__((ext_vector_type(4)));

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int PADB = 96;  // a tile that touches the bias's changing distances reaches at most 64 + 31 beyond them

struct LaParams {
    int B, H, Hk, G, Sq, Sk, D;
    int HG, Gr;  // row groups of the grid: Hk groups of G heads' rows packed together, or (bias) H groups of one head
    int causal, q_start;
    float scale, sc;  // sc = scale * log2(e): the softmax runs in base 2
    const int32_t *mask, *count;
    const void *Q[2], *K[2], *V[2], *dO, *O[2];
    void *Ow[2], *dQ, *dK, *dV;
    int64_t qb, kb, vb, ob, dob, dqb, dkb, dvb;  // elements between dialogs
    int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    float* lse;
    float* delta;   // [B][H][Sq] do . o, then [B][H][Sq] |do| (fp16)
    const void* table;  // [nb][H]
    const int32_t* map; // [2 maxd + 1]
    int nb, maxd;
    float drop_p, inv_keep;
    uint32_t thr;
    uint64_t seed, offset;
    int ns, nrt;    // splits of the contraction, row (key) tiles
    float *part, *ml, *part2, *tpart;
};

// ---- element types: how operands lie in memory, what multiplies them
template <bool F16_>
struct E16 {
    static constexpr bool F32 = false, F16 = F16_;
    static constexpr int EPC = 8;  // elements per 16-byte LDS chunk
    __device__ static uint4 load(const void* const* p, int64_t off) { return *reinterpret_cast<const uint4*>(static_cast<const u16*>(p[0]) + off); }
    __device__ static float to_f32(u16 x) { return F16 ? f16_to_f32(x) : bf16_to_f32(x); }
    __device__ static void store4(void* const* p, int64_t off, const float v[4]) {
        uint2 hi, lo;
        split4(v, hi, lo, F16);
        *reinterpret_cast<uint2*>(static_cast<u16*>(p[0]) + off) = hi;
        if (p[1]) *reinterpret_cast<uint2*>(static_cast<u16*>(p[1]) + off) = lo;
    }
    __device__ static float elem(const void* p, int64_t off) { return to_f32(static_cast<const u16*>(p)[off]); }
};
struct EF32 {
    static constexpr bool F32 = true, F16 = false;
    static constexpr int EPC = 4;
    __device__ static uint4 load(const void* const* p, int64_t off) { return *reinterpret_cast<const uint4*>(static_cast<const float*>(p[0]) + off); }
    __device__ static void store4(void* const* p, int64_t off, const float v[4]) {
        *reinterpret_cast<float4*>(static_cast<float*>(p[0]) + off) = make_float4(v[0], v[1], v[2], v[3]);
    }
    __device__ static float elem(const void* p, int64_t off) { return static_cast<const float*>(p)[off]; }
};
// fp32 arithmetic on split planes (value = hi + lo), results as planes
template <bool F16_>
struct EPlanes {
    static constexpr bool F32 = true, F16 = F16_;
    static constexpr int EPC = 4;
    __device__ static uint4 load(const void* const* p, int64_t off) {
        float a[4], b[4];
        unpack4(*reinterpret_cast<const uint2*>(static_cast<const u16*>(p[0]) + off), a, F16);
        unpack4(*reinterpret_cast<const uint2*>(static_cast<const u16*>(p[1]) + off), b, F16);
        const float4 s = make_float4(a[0] + b[0], a[1] + b[1], a[2] + b[2], a[3] + b[3]);
        return __builtin_bit_cast(uint4, s);
    }
    __device__ static void store4(void* const* p, int64_t off, const float v[4]) { E16<F16_>::store4(p, off, v); }
    __device__ static float elem(const void* p, int64_t off) { return static_cast<const float*>(p)[off]; }
};

// ---- LDS images [rows][DP] in 16-byte chunks, XOR-swizzled so that a column of chunks (MFMA A rows) and the transposing reads
// spread over the banks
template <int CH>
__device__ __forceinline__ int swz(int row) {
    if constexpr (CH == 8) return row & 7;
    else if constexpr (CH % 8 == 0) return ((row & 3) << 1) | ((row >> 2) & 1);
    else return (row >> 2) & 3;
}
template <int CH>
__device__ __forceinline__ int lds_off(int row, int ch) { return (row * CH + (ch ^ swz<CH>(row))) * 16; }

__device__ __forceinline__ v4s tr_read(const char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p); }

template <bool F16>
__device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// B operand fragments of one lane's row, the whole head dim: 16-bit: chunk 2 ks + h (8 elements); fp32: chunk 2 c + h (4)
template <class T, int DP>
struct Frag {
    static constexpr int N = DP / (2 * T::EPC);
    uint4 x[N];
    __device__ void load(const void* const* p, int64_t off, bool ok, int D, int h) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int col = (2 * c + h) * T::EPC;
            x[c] = make_uint4(0, 0, 0, 0);
            if (ok && col < D) x[c] = T::load(p, off + col);
        }
    }
};

// acc[32 rows of the image][32 lanes] += image[row0 ..][.] . frag over the head dim
template <class T, int DP>
__device__ __forceinline__ f32x16 dot_rows(const char* img, int row0, const Frag<T, DP>& f, int lane, f32x16 acc) {
    constexpr int CH = DP / T::EPC;
    const int row = row0 + (lane & 31), h = lane >> 5;
#pragma unroll
    for (int c = 0; c < Frag<T, DP>::N; ++c) {
        const uint4 a = *reinterpret_cast<const uint4*>(img + lds_off<CH>(row, 2 * c + h));
        if constexpr (T::F32) {
            const float4 af = __builtin_bit_cast(float4, a), bf = __builtin_bit_cast(float4, f.x[c]);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.x, bf.x, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.y, bf.y, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.z, bf.z, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.w, bf.w, acc, 0, 0, 0);
        } else {
            acc = mma32<T::F16>(a, f.x[c], acc);
        }
    }
    return acc;
}

// acc[dt][d = 32 dt + ..][lane] += image[row0 + k][d] * w[k][lane] over the 32 rows k: w is a 32x32 result in the C layout
template <class T, int DP>
__device__ __forceinline__ void add_cols(const char* img, int row0, const f32x16& w, int lane, f32x16 acc[DP / 32]) {
    constexpr int CH = DP / T::EPC;
    const int h = lane >> 5;
    if constexpr (T::F32) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = row0 + 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) {
                const int d = dt * 32 + (lane & 31);
                const float a = *reinterpret_cast<const float*>(img + lds_off<CH>(row, d >> 2) + (d & 3) * 4);
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w[r], acc[dt], 0, 0, 0);
            }
        }
    } else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        uint32_t pk[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const f2 v = {w[2 * r], w[2 * r + 1]};
            if constexpr (T::F16) {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                pk[r] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
            } else {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                pk[r] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2));
            }
        }
        const int i = lane & 15, dh = (lane >> 4) & 1;  // this lane's address in its 16-lane group's 4 x 16 block; which half of the 32 columns
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint4 b = make_uint4(pk[4 * s], pk[4 * s + 1], pk[4 * s + 2], pk[4 * s + 3]);
            const int ra = row0 + 16 * s + 4 * h + (i >> 2);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) {
                const int ch = dt * 4 + dh * 2 + ((i & 3) >> 1), sub = (i & 1) * 8;
                const v4s lo = tr_read(img + lds_off<CH>(ra, ch) + sub), hi = tr_read(img + lds_off<CH>(ra + 8, ch) + sub);
                const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
                acc[dt] = mma32<T::F16>(make_uint4(l2.x, l2.y, h2.x, h2.y), b, acc[dt]);
            }
        }
    }
}

// one operand's tile, global -> registers -> LDS image; rows at or past `n` (and masked ones) become zeros
template <class T, int DP, int ROWS>
struct Stage {
    static constexpr int CH = DP / T::EPC, NC = (ROWS * CH + 255) / 256;
    uint4 x[NC];
    __device__ __forceinline__ void load(const void* const* p, int64_t base, int64_t ld, int row0, int n, int D, int tid) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = tid + j * 256, row = c / CH, col = (c % CH) * T::EPC;
            x[j] = make_uint4(0, 0, 0, 0);
            if (row < ROWS && row0 + row < n && col < D) x[j] = T::load(p, base + (row0 + row) * ld + col);
        }
    }
    __device__ __forceinline__ void zero(const uint32_t keep[NC]) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (!keep[j]) x[j] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void store(char* img, int tid) const {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = tid + j * 256, row = c / CH;
            if (row < ROWS) *reinterpret_cast<uint4*>(img + lds_off<CH>(row, c % CH)) = x[j];
        }
    }
};

__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// neighbouring work items share keys and values: keep them on one XCD (workgroups go round the eight XCDs one by one)
__device__ __forceinline__ int xcd_order(int id, int n) {
    const int x = id & 7, q = n >> 3, r = n & 7;
    return x * q + min(x, r) + (id >> 3);
}

__device__ __forceinline__ int visible_end(const LaParams& p, int b) {
    int e = p.Sk;
    if (p.count) e = min(e, max(0, __builtin_amdgcn_readfirstlane(p.count[b])));
    return e;
}

// The bias as a function of the distance alone, for one head, in base-2 units: bv[d + maxd + PADB] for |d| <= maxd + PADB; outside
// [lo, hi] the buckets are those of the ends.  A bucket outside the table gives NaN.
struct Bias {
    float *v, left, right;
    int lo, hi;
};
template <class T>
__device__ __forceinline__ void bias_fill(const LaParams& p, int head, float* v, int tid) {
    const int n = 2 * p.maxd + 1 + 2 * PADB;
    for (int x = tid; x < n; x += 256) {
        const int t = p.map[min(max(x - PADB, 0), 2 * p.maxd)];
        v[x] = t >= 0 && t < p.nb ? T::elem(p.table, (int64_t)t * p.H + head) * LOG2E : __builtin_nanf("");
    }
}
// first and last distance whose bucket differs from that of the end on its side; every thread gets both (sh: 8 ints)
__device__ __forceinline__ void bias_range(const LaParams& p, int* sh, int tid, int& lo, int& hi) {
    const int a = p.map[0], z = p.map[2 * p.maxd];
    int l = p.maxd + 1, h = -p.maxd - 1;
    for (int x = tid; x <= 2 * p.maxd; x += 256) {
        const int t = p.map[x];
        if (t != a) l = min(l, x - p.maxd);
        if (t != z) h = max(h, x - p.maxd);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        l = min(l, __shfl_xor(l, o, 64));
        h = max(h, __shfl_xor(h, o, 64));
    }
    if ((tid & 63) == 0) {
        sh[tid >> 6] = l;
        sh[4 + (tid >> 6)] = h;
    }
    __syncthreads();
    lo = min(min(sh[0], sh[1]), min(sh[2], sh[3]));
    hi = max(max(sh[4], sh[5]), max(sh[6], sh[7]));
    // one bucket throughout (or two that meet): everything left of lo is the left end's, everything from lo on the right end's
    hi = max(hi, lo - 1);
    lo = min(lo, hi + 1);
}

// keep (1 / (1 - p)) or drop (0) of the 4 probabilities of keys j0 .. j0 + 3 (j0 % 4 == 0) of one row: the stream of
// didi_attention_train_forward: element (b, h, i, j) is dropped iff word j & 3 of Philox(offset + ((b H + h) Sq + i) ceil(Sk / 4) + j / 4) < p 2^32
__device__ __forceinline__ void drop4(const LaParams& p, uint64_t row, int j0, float k[4]) {
    uint32_t w[4];
    philox4x32_10(p.offset + row * (uint64_t)((p.Sk + 3) >> 2) + (uint64_t)(j0 >> 2), p.seed, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = w[e] < p.thr ? 0.f : p.inv_keep;
}

// ------------------------------------------------------------------ forward
// WK = 1: a workgroup owns 128 rows, its four waves 32 each, over tiles of BN keys.  WK = 4: 32 rows, the four waves take a quarter
// of every key tile each and join at the end (few rows: one token per dialog).
template <class T, int DP, int WK>
struct FwdCfg {
    static constexpr int NT = WK == 4 ? 1 : (T::F32 ? 1 : 2);
    static constexpr int BN = WK == 4 ? 128 : 32 * NT;
    static constexpr int ROWS = WK == 4 ? 32 : 128;
    static constexpr int IMG = BN * DP * (16 / T::EPC);  // bytes of one operand's image
    static constexpr int NBUF = 4 * IMG <= 128 * 1024 ? 2 : 1;
    static constexpr int LDS = 2 * NBUF * IMG;
    static_assert(WK == 1 || LDS >= 4 * 32 * (DP + 4) * 4 + 4 * 32 * 8, "the join of the waves reuses the images");
};

template <class T, int DP, int WK>
__global__ void __launch_bounds__(256, T::F32 ? 1 : 2) la_forward(LaParams p) {
    using C = FwdCfg<T, DP, WK>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    if constexpr (T::F16) f16_saturate_mode();
    int w = xcd_order(blockIdx.x, gridDim.x);
    const int split = w % p.ns;
    w /= p.ns;
    const int rt = w % p.nrt;
    w /= p.nrt;
    const int hg = w % p.HG, b = w / p.HG, head0 = hg * p.Gr, kvh = head0 / p.G;
    const int R = p.Gr * p.Sq, rbase = rt * C::ROWS, rw = rbase + (WK == 1 ? wave * 32 : 0);
    const int r = rw + (lane & 31);
    const bool rok = r < R;
    const int g = rok ? r / p.Sq : 0, i = rok ? r - g * p.Sq : 0, head = head0 + g, pos = p.q_start + i;
    const uint64_t rowid = ((uint64_t)b * p.H + head) * p.Sq + i;
    int kend = visible_end(p, b);
    if (p.causal) {
        const int last = min(R, rbase + C::ROWS) - 1;
        kend = min(kend, p.q_start + (rbase / p.Sq == last / p.Sq ? last % p.Sq : p.Sq - 1) + 1);
    }
    const int tiles = (kend + C::BN - 1) / C::BN, per = (tiles + p.ns - 1) / p.ns;
    const int t0 = split * per, t1 = min(tiles, t0 + per);

    Frag<T, DP> q;
    q.load(p.Q, (int64_t)b * p.qb + (int64_t)i * p.ldq + head * p.D, rok, p.D, h);
    float* bv = reinterpret_cast<float*>(smem + C::LDS);
    const bool biased = p.table != nullptr;
    int blo = 0, bhi = -1;
    if (biased) {
        bias_fill<T>(p, head0, bv, tid);
        bias_range(p, reinterpret_cast<int*>(bv + 2 * p.maxd + 1 + 2 * PADB), tid, blo, bhi);
    }

    f32x16 o[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    float m = -INFINITY, l = 0.f;  // maximum in units of t (base 2: biased) or of q . k; l: this lane's half of the row's sum
    const float mul = biased ? 1.f : p.sc;

    const int64_t kbase = (int64_t)b * p.kb + kvh * p.D, vbase = (int64_t)b * p.vb + kvh * p.D;
    const int32_t* mrow = p.mask ? p.mask + (int64_t)b * p.Sk : nullptr;
    Stage<T, DP, C::BN> sk, sv;
    uint32_t keep[Stage<T, DP, C::BN>::NC];
    auto fetch = [&](int t) {
        sk.load(p.K, kbase, p.ldk, t * C::BN, kend, p.D, tid);
        sv.load(p.V, vbase, p.ldv, t * C::BN, kend, p.D, tid);
        if (mrow) {
#pragma unroll
            for (int j = 0; j < Stage<T, DP, C::BN>::NC; ++j) {
                const int key = t * C::BN + (tid + j * 256) / Stage<T, DP, C::BN>::CH;
                keep[j] = key < kend ? (uint32_t)mrow[key] : 0u;
            }
        }
    };
    auto put = [&](int buf) {
        if (mrow) {
            sk.zero(keep);
            sv.zero(keep);
        }
        sk.store(smem + buf * 2 * C::IMG, tid);
        sv.store(smem + buf * 2 * C::IMG + C::IMG, tid);
    };
    if (t0 < t1) {
        fetch(t0);
        put(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = C::NBUF == 2 ? (t - t0) & 1 : 0;
        const char *Ks = smem + buf * 2 * C::IMG, *Vs = Ks + C::IMG;
        if (t + 1 < t1) fetch(t + 1);
        const int krow = WK == 4 ? wave * 32 : 0, k0 = t * C::BN + krow;
        // which of the wave's keys this lane's row sees
        uint64_t bits = low_bits(kend - k0);
        if (mrow) bits &= __ballot(lane < 32 * C::NT && k0 + lane < kend && mrow[k0 + lane] != 0);
        if constexpr (C::NT == 1) bits &= 0xffffffffull;
        constexpr uint64_t ALL = C::NT == 1 ? 0xffffffffull : ~0ull;
        bool full = bits == ALL;
        if (bits) {
            if (p.causal) {
                const uint64_t mine = low_bits(pos - k0 + 1) & ALL;
                full = full && __all(mine == ALL);
                bits &= mine;
            }
            f32x16 s[C::NT];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                f32x16 z;
#pragma unroll
                for (int e = 0; e < 16; ++e) z[e] = 0.f;
                s[nt] = dot_rows<T, DP>(Ks, krow + nt * 32, q, lane, z);
            }
            if (biased) {
                const int pmin = p.q_start + rw, dmin = k0 - pmin - 31, dmax = k0 + 32 * C::NT - 1 - pmin;
                if (dmax < blo || dmin > bhi) {
                    const float c = dmax < blo ? bv[0] : bv[2 * p.maxd + 2 * PADB];
#pragma unroll
                    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[nt][e] = fmaf(s[nt][e], p.sc, c);
                } else {
                    const float* at = bv + (k0 - (p.q_start + r) + p.maxd + PADB + 4 * h);
#pragma unroll
                    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[nt][e] = fmaf(s[nt][e], p.sc, at[nt * 32 + 8 * (e >> 2) + (e & 3)]);
                }
            }
            if (!full) {
                const uint64_t mine = bits >> (4 * h);
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!((mine >> (nt * 32 + 8 * (e >> 2) + (e & 3))) & 1)) s[nt][e] = -INFINITY;
            }
            float top = s[0][0];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, s[nt][e]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m)) {
                const float mn = fmaxf(m, top);
                const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * mul);
                m = mn;
                l *= a;
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[dt][e] *= a;
            }
            const float sub = m == -INFINITY ? 0.f : -m * mul;
            float ls = 0.f;
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[nt][e] = __builtin_amdgcn_exp2f(fmaf(s[nt][e], mul, sub));
                    ls += s[nt][e];
                }
            l += ls;
            if (p.drop_p > 0.f) {
#pragma unroll
                for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
                    for (int gq = 0; gq < 4; ++gq) {
                        float k[4];
                        drop4(p, rowid, k0 + nt * 32 + 8 * gq + 4 * h, k);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[nt][4 * gq + e] *= k[e];
                    }
            }
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) add_cols<T, DP>(Vs, krow + nt * 32, s[nt], lane, o);
        }
        if constexpr (C::NBUF == 1) __syncthreads();
        if (t + 1 < t1) put(C::NBUF == 2 ? buf ^ 1 : 0);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    const float m2 = m * mul;  // base-2 maximum

    const int64_t rows_all = (int64_t)p.B * p.H * p.Sq;
    if constexpr (WK == 1) {
        if (!rok) return;
        const float inv = p.ns > 1 ? 1.f : l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int d = dt * 32 + gq * 8 + 4 * h;
                if (d >= p.D) continue;
                const float v[4] = {o[dt][4 * gq] * inv, o[dt][4 * gq + 1] * inv, o[dt][4 * gq + 2] * inv, o[dt][4 * gq + 3] * inv};
                if (p.ns > 1) *reinterpret_cast<float4*>(p.part + ((int64_t)split * rows_all + rowid) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
                else T::store4(p.Ow, (int64_t)b * p.ob + (int64_t)i * p.ldo + head * p.D + d, v);
            }
        if (h == 0) {
            if (p.ns > 1) *reinterpret_cast<float2*>(p.ml + ((int64_t)split * rows_all + rowid) * 2) = make_float2(m2, l);
            else if (p.lse) p.lse[rowid] = l > 0.f ? (m2 + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
        }
    } else {
        // join the four waves: O^T to LDS as [wave][row][d], maxima and sums beside it
        constexpr int LD = DP + 4;
        float* ox = reinterpret_cast<float*>(smem);
        float2* mx = reinterpret_cast<float2*>(ox + 4 * 32 * LD);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq)
                *reinterpret_cast<float4*>(ox + (wave * 32 + (lane & 31)) * LD + dt * 32 + gq * 8 + 4 * h) =
                    make_float4(o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]);
        if (h == 0) mx[wave * 32 + (lane & 31)] = make_float2(m2, l);
        __syncthreads();
        for (int x = tid; x < 32 * (DP / 4); x += 256) {
            const int row = x / (DP / 4), d = x % (DP / 4) * 4, rr = rbase + row;
            if (rr >= R || d >= p.D) continue;
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, mx[k * 32 + row].x);
            float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 e = mx[k * 32 + row];
                if (!(e.y > 0.f)) continue;
                const float a = __builtin_amdgcn_exp2f(e.x - top);
                sum += a * e.y;
                const float4 ov = *reinterpret_cast<const float4*>(ox + (k * 32 + row) * LD + d);
                v[0] = fmaf(a, ov.x, v[0]);
                v[1] = fmaf(a, ov.y, v[1]);
                v[2] = fmaf(a, ov.z, v[2]);
                v[3] = fmaf(a, ov.w, v[3]);
            }
            const int gg = rr / p.Sq, ii = rr - gg * p.Sq, hd = head0 + gg;
            const int64_t id = ((int64_t)b * p.H + hd) * p.Sq + ii;
            if (p.ns > 1) {
                *reinterpret_cast<float4*>(p.part + ((int64_t)split * rows_all + id) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) *reinterpret_cast<float2*>(p.ml + ((int64_t)split * rows_all + id) * 2) = make_float2(top, sum);
            } else {
                const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= inv;
                T::store4(p.Ow, (int64_t)b * p.ob + (int64_t)ii * p.ldo + hd * p.D + d, v);
                if (d == 0 && p.lse) p.lse[id] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
            }
        }
    }
}

// joins the splits of the forward: one thread per four head-dim elements of a row
template <class T>
__global__ void __launch_bounds__(256) la_join(LaParams p) {
    const int64_t rows = (int64_t)p.B * p.H * p.Sq, x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d4 = p.D / 4;
    const int64_t row = x / d4;
    if (row >= rows) return;
    const int d = (int)(x - row * d4) * 4;
    float top = -INFINITY;
    for (int s = 0; s < p.ns; ++s) {
        const float2 e = *reinterpret_cast<const float2*>(p.ml + (s * rows + row) * 2);
        if (e.y > 0.f) top = fmaxf(top, e.x);
    }
    float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.ns; ++s) {
        const float2 e = *reinterpret_cast<const float2*>(p.ml + (s * rows + row) * 2);
        const float4 o = *reinterpret_cast<const float4*>(p.part + (s * rows + row) * p.D + d);
        if (!(e.y > 0.f)) continue;
        const float a = __builtin_amdgcn_exp2f(e.x - top);
        sum = fmaf(a, e.y, sum);
        v[0] = fmaf(a, o.x, v[0]);
        v[1] = fmaf(a, o.y, v[1]);
        v[2] = fmaf(a, o.z, v[2]);
        v[3] = fmaf(a, o.w, v[3]);
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= inv;
    const int i = (int)(row % p.Sq);
    const int64_t bh = row / p.Sq;
    T::store4(p.Ow, bh / p.H * p.ob + (int64_t)i * p.ldo + bh % p.H * p.D + d, v);
    if (d == 0 && p.lse) p.lse[row] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
}

// ------------------------------------------------------------------ backward: dQ, D = do . o, and the sums of ds by distance
// fp16: ds is scaled by a power of two before it is rounded to 16 bits, so that small gradients keep their bits: 64 / |do_i| per row here
// (undone at the end: the lane owns the row), 64 / max_i |do_i| of the head in la_backward_kv.  |ds| <= 2 |do| max|v|, so nothing
// saturates below |v| = 512, and probabilities down to 1e-6 of a row stay normal numbers.
__device__ __forceinline__ float pow2_scale(float norm) {
    if (!(norm > 0.f) || !(norm < INFINITY)) return 1.f;
    const int e = (int)((__builtin_bit_cast(uint32_t, norm) >> 23) & 0xff) - 127;  // norm >= 2^e
    return __builtin_bit_cast(float, (uint32_t)(127 + min(max(5 - e, -100), 100)) << 23);
}

template <class T, int DP>
struct BwdQCfg {
    static constexpr int NT = T::F32 ? 1 : 2, BN = 32 * NT;
    static constexpr int IMG = BN * DP * (16 / T::EPC);
    static constexpr int LDS = 4 * IMG;  // two buffers of K and V
};

// where the table's gradient is accumulated: one array of distances per wave and lane half (each address is then touched at most once
// per instruction, so the LDS adds have one order), index d + maxd + PADB
__device__ __forceinline__ int dist_len(int maxd) { return 2 * maxd + 1 + 2 * PADB; }

template <class T, int DP>
__global__ void __launch_bounds__(256, T::F32 ? 1 : 2) la_backward_q(LaParams p) {
    using C = BwdQCfg<T, DP>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    if constexpr (T::F16) f16_saturate_mode();
    int w = xcd_order(blockIdx.x, gridDim.x);
    const int wg = w;
    const int split = w % p.ns;
    w /= p.ns;
    const int rt = w % p.nrt;
    w /= p.nrt;
    const int hg = w % p.HG, b = w / p.HG, head0 = hg * p.Gr, kvh = head0 / p.G;
    const int R = p.Gr * p.Sq, rbase = rt * 128, rw = rbase + wave * 32;
    const int r = rw + (lane & 31);
    const bool rok = r < R;
    const int g = rok ? r / p.Sq : 0, i = rok ? r - g * p.Sq : 0, head = head0 + g, pos = p.q_start + i;
    const int64_t rowid = ((int64_t)b * p.H + head) * p.Sq + i;
    int kend = visible_end(p, b);
    if (p.causal) {
        const int last = min(R, rbase + 128) - 1;
        kend = min(kend, p.q_start + (rbase / p.Sq == last / p.Sq ? last % p.Sq : p.Sq - 1) + 1);
    }
    const int tiles = (kend + C::BN - 1) / C::BN, per = (tiles + p.ns - 1) / p.ns;
    const int t0 = split * per, t1 = min(tiles, t0 + per);

    Frag<T, DP> q, go;
    q.load(p.Q, (int64_t)b * p.qb + (int64_t)i * p.ldq + head * p.D, rok, p.D, h);
    const void* dop[2] = {p.dO, nullptr};
    go.load(dop, (int64_t)b * p.dob + (int64_t)i * p.lddo + head * p.D, rok, p.D, h);
    float delta = 0.f, norm = 0.f;
    {
        const int64_t oo = (int64_t)b * p.ob + (int64_t)i * p.ldo + head * p.D;
        Frag<T, DP> o;
        o.load(p.O, oo, rok, p.D, h);
#pragma unroll
        for (int c = 0; c < Frag<T, DP>::N; ++c) {
            if constexpr (T::F32) {
                const float4 a = __builtin_bit_cast(float4, o.x[c]), e = __builtin_bit_cast(float4, go.x[c]);
                delta = fmaf(a.x, e.x, fmaf(a.y, e.y, fmaf(a.z, e.z, fmaf(a.w, e.w, delta))));
            } else {
                const uint32_t a[4] = {o.x[c].x, o.x[c].y, o.x[c].z, o.x[c].w}, e[4] = {go.x[c].x, go.x[c].y, go.x[c].z, go.x[c].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float e0 = T::to_f32((u16)e[k]), e1 = T::to_f32((u16)(e[k] >> 16));
                    delta = fmaf(T::to_f32((u16)a[k]), e0, fmaf(T::to_f32((u16)(a[k] >> 16)), e1, delta));
                    norm = fmaf(e0, e0, fmaf(e1, e1, norm));
                }
            }
        }
        if constexpr (!T::F32) {
            if (p.O[1]) {  // the output's remainder: the sums of ds by distance cancel, so D wants more than the output's 8 or 11 bits
                const void* lo[2] = {p.O[1], nullptr};
                o.load(lo, oo, rok, p.D, h);
#pragma unroll
                for (int c = 0; c < Frag<T, DP>::N; ++c) {
                    const uint32_t a[4] = {o.x[c].x, o.x[c].y, o.x[c].z, o.x[c].w}, e[4] = {go.x[c].x, go.x[c].y, go.x[c].z, go.x[c].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        delta = fmaf(T::to_f32((u16)a[k]), T::to_f32((u16)e[k]), fmaf(T::to_f32((u16)(a[k] >> 16)), T::to_f32((u16)(e[k] >> 16)), delta));
                }
            }
        }
        delta += __shfl_xor(delta, 32, 64);
        norm += __shfl_xor(norm, 32, 64);
    }
    norm = __builtin_amdgcn_sqrtf(norm);
    if (split == 0 && rok && h == 0) {
        p.delta[rowid] = delta;
        if constexpr (T::F16) p.delta[(int64_t)p.B * p.H * p.Sq + rowid] = norm;
    }
    const float fs = T::F16 ? pow2_scale(norm) : 1.f;
    const float lse = rok ? p.lse[rowid] : -INFINITY;
    const float sub = lse == -INFINITY ? -INFINITY : -lse * LOG2E;  // a row that sees nothing: p = exp2(-inf) = 0

    float* bv = reinterpret_cast<float*>(smem + C::LDS);
    const bool biased = p.table != nullptr;
    int blo = 0, bhi = -1;
    const int len = dist_len(p.maxd);
    float* acc_d = bv + len + 8;  // [4 waves][2 halves][len]
    if (biased) {
        bias_fill<T>(p, head0, bv, tid);
        for (int x = tid; x < 8 * len; x += 256) acc_d[x] = 0.f;
        bias_range(p, reinterpret_cast<int*>(bv + len), tid, blo, bhi);
    }
    float* mine_d = acc_d + (wave * 2 + h) * len;
    float far_l = 0.f, far_r = 0.f;

    f32x16 dq[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[dt][e] = 0.f;

    const int64_t kbase = (int64_t)b * p.kb + kvh * p.D, vbase = (int64_t)b * p.vb + kvh * p.D;
    const int32_t* mrow = p.mask ? p.mask + (int64_t)b * p.Sk : nullptr;
    Stage<T, DP, C::BN> sk, sv;
    uint32_t keep[Stage<T, DP, C::BN>::NC];
    auto fetch = [&](int t) {
        sk.load(p.K, kbase, p.ldk, t * C::BN, kend, p.D, tid);
        sv.load(p.V, vbase, p.ldv, t * C::BN, kend, p.D, tid);
        if (mrow) {
#pragma unroll
            for (int j = 0; j < Stage<T, DP, C::BN>::NC; ++j) {
                const int key = t * C::BN + (tid + j * 256) / Stage<T, DP, C::BN>::CH;
                keep[j] = key < kend ? (uint32_t)mrow[key] : 0u;
            }
        }
    };
    auto put = [&](int buf) {
        if (mrow) {
            sk.zero(keep);
            sv.zero(keep);
        }
        sk.store(smem + buf * 2 * C::IMG, tid);
        sv.store(smem + buf * 2 * C::IMG + C::IMG, tid);
    };
    if (t0 < t1) {
        fetch(t0);
        put(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, k0 = t * C::BN;
        const char *Ks = smem + buf * 2 * C::IMG, *Vs = Ks + C::IMG;
        if (t + 1 < t1) fetch(t + 1);
        uint64_t bits = low_bits(kend - k0);
        if (mrow) bits &= __ballot(lane < C::BN && k0 + lane < kend && mrow[k0 + lane] != 0);
        constexpr uint64_t ALL = C::NT == 1 ? 0xffffffffull : ~0ull;
        bits &= ALL;
        bool full = bits == ALL;
        if (bits) {
            if (p.causal) {
                const uint64_t mine = low_bits(pos - k0 + 1) & ALL;
                full = full && __all(mine == ALL);
                bits &= mine;
            }
            const int pmin = p.q_start + rw, dmin = k0 - pmin - 31, dmax = k0 + C::BN - 1 - pmin;
            const bool left = dmax < blo, near = biased && !left && dmin <= bhi;
            const float fc = biased ? (left ? bv[0] : bv[len - 1]) : 0.f;
            const int at = k0 - (p.q_start + r) + p.maxd + PADB + 4 * h;
            const uint64_t mine = bits >> (4 * h);
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                f32x16 s, dp;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
                s = dot_rows<T, DP>(Ks, nt * 32, q, lane, s);
                dp = dot_rows<T, DP>(Vs, nt * 32, go, lane, dp);
                if (near) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.sc, bv[at + nt * 32 + 8 * (e >> 2) + (e & 3)] + sub));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.sc, fc + sub));
                }
                if (!full) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!((mine >> (nt * 32 + 8 * (e >> 2) + (e & 3))) & 1)) s[e] = 0.f;
                }
                if (p.drop_p > 0.f) {
#pragma unroll
                    for (int gq = 0; gq < 4; ++gq) {
                        float k[4];
                        drop4(p, (uint64_t)rowid, k0 + nt * 32 + 8 * gq + 4 * h, k);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dp[4 * gq + e] *= k[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= dp[e] - delta;
                if (biased && p.tpart) {
                    if (near) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) atomicAdd(&mine_d[at + nt * 32 + 8 * (e >> 2) + (e & 3)], s[e]);
                    } else {
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) sum += s[e];
                        if (left) far_l += sum;
                        else far_r += sum;
                    }
                }
                if constexpr (T::F16) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] *= fs;
                }
                add_cols<T, DP>(Ks, nt * 32, s, lane, dq);
            }
        }
        if (t + 1 < t1) put(buf ^ 1);
        __syncthreads();
    }
    if (rok) {
        const float out = p.scale / fs;
        void* dqp[2] = {p.dQ, nullptr};
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int d = dt * 32 + gq * 8 + 4 * h;
                if (d >= p.D) continue;
                const float v[4] = {dq[dt][4 * gq] * out, dq[dt][4 * gq + 1] * out, dq[dt][4 * gq + 2] * out, dq[dt][4 * gq + 3] * out};
                if (p.ns > 1) *reinterpret_cast<float4*>(p.part + ((int64_t)split * p.B * p.H * p.Sq + rowid) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
                else T::store4(dqp, (int64_t)b * p.dqb + (int64_t)i * p.lddq + head * p.D + d, v);
            }
    }
    if (biased && p.tpart) {
        // this workgroup's sums by distance: the eight arrays joined in a fixed order; what lies beyond the map's ends joins the far tiles
        float* fx = bv;  // the bias is no longer needed
        far_l = wave_sum(far_l);
        far_r = wave_sum(far_r);
        __syncthreads();
        if (lane == 0) {
            fx[wave] = far_l;
            fx[4 + wave] = far_r;
        }
        for (int x = tid; x < len; x += 256) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += acc_d[k * len + x];
            acc_d[x] = sum;
        }
        __syncthreads();
        const int nd = 2 * p.maxd + 1;
        float* out = p.tpart + (int64_t)wg * (nd + 2);
        for (int x = tid; x < nd; x += 256) out[x] = acc_d[PADB + x];
        if (wave < 2) {
            float sum = 0.f;
            for (int x = lane; x < PADB; x += 64) sum += acc_d[wave == 0 ? x : len - PADB + x];
            sum = wave_sum(sum);
            if (lane == 0) out[nd + wave] = sum + fx[4 * wave] + fx[4 * wave + 1] + fx[4 * wave + 2] + fx[4 * wave + 3];
        }
    }
}

// dtable[t][h] from the sums by distance of `parts` workgroups per (dialog, head) -- tpart [B][H][parts][2 maxd + 1 distances, left, right] --
// added in a fixed order; one workgroup per head
template <class T>
__global__ void __launch_bounds__(1024) la_table_sum(const float* tpart, const int32_t* map, int B, int H, int parts, int nb, int maxd, void* out) {
    extern __shared__ float dist[];  // [4][nd + 2]
    const int h = blockIdx.x, nd = 2 * maxd + 1, n = nd + 2, tid = threadIdx.x, grp = tid >> 8, total = B * parts;
    for (int x = tid & 255; x < n; x += 256) {
        float sum = 0.f;
        for (int k = grp; k < total; k += 4) {
            const int b = k / parts;
            sum += tpart[(((int64_t)b * H + h) * parts + (k - b * parts)) * n + x];
        }
        dist[grp * n + x] = sum;
    }
    __syncthreads();
    for (int x = tid; x < n; x += 1024) dist[x] = (dist[x] + dist[n + x]) + (dist[2 * n + x] + dist[3 * n + x]);
    __syncthreads();
    // one wave per bucket: its lanes take the distances in turn
    const int lane = tid & 63;
    for (int t = tid >> 6; t < nb; t += 16) {
        float sum = 0.f;
        for (int x = lane; x < nd; x += 64)
            if (map[x] == t) sum += dist[x];
        if (lane == 0 && map[0] == t) sum += dist[nd];
        if (lane == 1 && map[2 * maxd] == t) sum += dist[nd + 1];
        sum = wave_sum(sum);
        if (lane == 0) {
            if constexpr (T::F32) static_cast<float*>(out)[(int64_t)t * H + h] = sum;
            else static_cast<u16*>(out)[(int64_t)t * H + h] = T::F16 ? f16_bits(sum) : bf16_bits(sum);
        }
    }
}

// out row = sum of the splits' partial rows
template <class T>
__global__ void __launch_bounds__(256) la_sum_parts(const float* part, int ns, int64_t rows, int per_bh, int heads, int D, void* out, int64_t batch, int ld) {
    const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d4 = D / 4;
    const int64_t row = x / d4;
    if (row >= rows) return;
    const int d = (int)(x - row * d4) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ns; ++s) {
        const float4 a = *reinterpret_cast<const float4*>(part + (s * rows + row) * D + d);
        v[0] += a.x;
        v[1] += a.y;
        v[2] += a.z;
        v[3] += a.w;
    }
    const int64_t bh = row / per_bh;
    void* o[2] = {out, nullptr};
    T::store4(o, bh / heads * batch + (row % per_bh) * ld + bh % heads * D + d, v);
}

// ------------------------------------------------------------------ backward: dK, dV
// A workgroup owns 128 keys of one key head, its waves 32 each (lane = key: K and V rows live in registers); it walks tiles of BQ rows of
// Q and dO of every head of the group.
template <class T, int DP>
struct BwdKCfg {
    static constexpr int NT = T::F32 ? 1 : 2, BQ = 32 * NT;
    static constexpr int IMG = BQ * DP * (16 / T::EPC);
    static constexpr int LDS = 4 * IMG + 4 * BQ * 4;  // two buffers of Q, dO; -lse and D of their rows
};

template <class T, int DP>
__global__ void __launch_bounds__(256, T::F32 || DP > 64 ? 1 : 2) la_backward_kv(LaParams p) {
    using C = BwdKCfg<T, DP>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    if constexpr (T::F16) f16_saturate_mode();
    int w = xcd_order(blockIdx.x, gridDim.x);
    const int split = w % p.ns;
    w /= p.ns;
    const int kt = w % p.nrt;
    w /= p.nrt;
    const int kvh = w % p.Hk, b = w / p.Hk;
    const int kw = kt * 128 + wave * 32, key = kw + (lane & 31);
    const int kend = visible_end(p, b);
    const bool vis = key < kend && (!p.mask || p.mask[(int64_t)b * p.Sk + key] != 0);
    const int64_t kvrow = (int64_t)b * p.kb + (int64_t)key * p.ldk + kvh * p.D, vrow = (int64_t)b * p.vb + (int64_t)key * p.ldv + kvh * p.D;

    Frag<T, DP> kf, vf;
    kf.load(p.K, kvrow, vis, p.D, h);
    vf.load(p.V, vrow, vis, p.D, h);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[dt][e] = dv[dt][e] = 0.f;

    float* rows_f = reinterpret_cast<float*>(smem + 4 * C::IMG);  // [2 buffers][-lse log2(e) | D][BQ]
    float* bv = reinterpret_cast<float*>(smem + C::LDS);
    const bool biased = p.table != nullptr;
    const int len = dist_len(p.maxd);
    int blo = 0, bhi = -1;
    if (biased) bias_range(p, reinterpret_cast<int*>(bv + len), tid, blo, bhi);
    float fs = 1.f;
    if constexpr (T::F16) {
        float top = 0.f;
        const float* norms = p.delta + (int64_t)p.B * p.H * p.Sq + ((int64_t)b * p.H + kvh * p.G) * p.Sq;
        for (int x = tid; x < p.G * p.Sq; x += 256) top = fmaxf(top, norms[x]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        if (lane == 0) rows_f[wave] = top;
        __syncthreads();
        fs = pow2_scale(fmaxf(fmaxf(rows_f[0], rows_f[1]), fmaxf(rows_f[2], rows_f[3])));
        __syncthreads();
    }

    const int qt0 = p.causal ? min(max(0, kt * 128 - p.q_start), p.Sq) / C::BQ : 0, nq = (p.Sq + C::BQ - 1) / C::BQ - qt0;
    const int tiles = kt * 128 < kend ? p.G * max(nq, 0) : 0, per = (tiles + p.ns - 1) / p.ns;
    const int t0 = split * per, t1 = min(tiles, t0 + per);
    Stage<T, DP, C::BQ> sq, sg;
    float row_c = 0.f;
    const void* dop[2] = {p.dO, nullptr};
    auto fetch = [&](int t) {
        const int head = kvh * p.G + t / nq, i0 = (qt0 + t % nq) * C::BQ;
        sq.load(p.Q, (int64_t)b * p.qb + head * p.D, p.ldq, i0, p.Sq, p.D, tid);
        sg.load(dop, (int64_t)b * p.dob + head * p.D, p.lddo, i0, p.Sq, p.D, tid);
        if (tid < 2 * C::BQ) {
            const int i = i0 + (tid < C::BQ ? tid : tid - C::BQ);
            const int64_t rowid = ((int64_t)b * p.H + head) * p.Sq + i;
            if (tid < C::BQ) {  // rows behind the last and rows that see nothing: p = exp2(-inf) = 0
                const float x = i < p.Sq ? p.lse[rowid] : -INFINITY;
                row_c = x == -INFINITY ? -INFINITY : -x * LOG2E;
            } else {
                row_c = i < p.Sq ? p.delta[rowid] : 0.f;
            }
        }
    };
    auto put = [&](int buf) {
        sq.store(smem + buf * 2 * C::IMG, tid);
        sg.store(smem + buf * 2 * C::IMG + C::IMG, tid);
        if (tid < 2 * C::BQ) rows_f[buf * 2 * C::BQ + tid] = row_c;
    };
    if (t0 < t1) {
        fetch(t0);
        put(0);
    }
    __syncthreads();
    int gcur = -1;
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, g = t / nq, i0 = (qt0 + t % nq) * C::BQ, head = kvh * p.G + g;
        const char *Qs = smem + buf * 2 * C::IMG, *Gs = Qs + C::IMG;
        const float* rc = rows_f + buf * 2 * C::BQ;
        if (biased && g != gcur) {  // another head of the group: its bias
            bias_fill<T>(p, head, bv, tid);
            __syncthreads();
            gcur = g;
        }
        if (t + 1 < t1) fetch(t + 1);
        // a wave none of whose keys is seen by the tile's last row has nothing to add
        if (!p.causal || kw <= p.q_start + min(i0 + C::BQ, p.Sq) - 1) {
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                const int i1 = i0 + nt * 32;
                f32x16 s, dp;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
                s = dot_rows<T, DP>(Qs, nt * 32, kf, lane, s);
                dp = dot_rows<T, DP>(Gs, nt * 32, vf, lane, dp);
                const int p0 = p.q_start + i1, dmin = kw - p0 - 31, dmax = kw + 31 - p0;
                const bool near = biased && dmax >= blo && dmin <= bhi;
                const float fc = vis ? (biased ? (dmax < blo ? bv[0] : bv[len - 1]) : 0.f) : -INFINITY;
                const int at = key - p0 + p.maxd + PADB - 4 * h;
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const int q0 = nt * 32 + 8 * gq + 4 * h;
                    const float4 l4 = *reinterpret_cast<const float4*>(rc + q0);
                    const float ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float c = near ? (vis ? bv[at - 8 * gq - e] : -INFINITY) : fc;
                        s[4 * gq + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * gq + e], p.sc, c + ls[e]));
                    }
                }
                if (p.causal && kw + 31 > p0) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (key > p0 + 8 * (e >> 2) + 4 * h + (e & 3)) s[e] = 0.f;
                }
                f32x16 ds;
                if (p.drop_p > 0.f) {
                    const int t4 = lane & 3;
#pragma unroll
                    for (int gq = 0; gq < 4; ++gq) {
                        // lane t of a quad (four neighbouring keys: one Philox counter) draws for row 8 gq + 4 h + t; word t of row e
                        // comes from lane e
                        const int i = i1 + 8 * gq + 4 * h + t4;
                        float k[4];
                        drop4(p, ((uint64_t)b * p.H + head) * p.Sq + i, key & ~3, k);
                        float mk[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int src = (lane & ~3) | e;
                            const float w0 = __shfl(k[0], src, 64), w1 = __shfl(k[1], src, 64), w2 = __shfl(k[2], src, 64), w3 = __shfl(k[3], src, 64);
                            mk[e] = t4 == 0 ? w0 : t4 == 1 ? w1 : t4 == 2 ? w2 : w3;
                        }
                        const float4 d4 = *reinterpret_cast<const float4*>(rc + C::BQ + nt * 32 + 8 * gq + 4 * h);
                        const float dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ds[4 * gq + e] = s[4 * gq + e] * fmaf(dp[4 * gq + e], mk[e], -dl[e]);
                            s[4 * gq + e] *= mk[e];
                        }
                    }
                } else {
#pragma unroll
                    for (int gq = 0; gq < 4; ++gq) {
                        const float4 d4 = *reinterpret_cast<const float4*>(rc + C::BQ + nt * 32 + 8 * gq + 4 * h);
                        const float dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) ds[4 * gq + e] = s[4 * gq + e] * (dp[4 * gq + e] - dl[e]);
                    }
                }
                if constexpr (T::F16) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) ds[e] *= fs;
                }
                add_cols<T, DP>(Gs, nt * 32, s, lane, dv);
                add_cols<T, DP>(Qs, nt * 32, ds, lane, dk);
            }
        }
        if (t + 1 < t1) put(buf ^ 1);
        __syncthreads();
    }
    if (key >= p.Sk) return;
    const float out = p.scale / fs;
    void *dkp[2] = {p.dK, nullptr}, *dvp[2] = {p.dV, nullptr};
    const int64_t rows = (int64_t)p.B * p.Hk * p.Sk, row = ((int64_t)b * p.Hk + kvh) * p.Sk + key;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
            const int d = dt * 32 + gq * 8 + 4 * h;
            if (d >= p.D) continue;
            const float a[4] = {dk[dt][4 * gq] * out, dk[dt][4 * gq + 1] * out, dk[dt][4 * gq + 2] * out, dk[dt][4 * gq + 3] * out};
            const float c[4] = {dv[dt][4 * gq], dv[dt][4 * gq + 1], dv[dt][4 * gq + 2], dv[dt][4 * gq + 3]};
            if (p.ns > 1) {
                *reinterpret_cast<float4*>(p.part + ((int64_t)split * rows + row) * p.D + d) = make_float4(a[0], a[1], a[2], a[3]);
                *reinterpret_cast<float4*>(p.part2 + ((int64_t)split * rows + row) * p.D + d) = make_float4(c[0], c[1], c[2], c[3]);
            } else {
                T::store4(dkp, (int64_t)b * p.dkb + (int64_t)key * p.lddk + kvh * p.D + d, a);
                T::store4(dvp, (int64_t)b * p.dvb + (int64_t)key * p.lddv + kvh * p.D + d, c);
            }
        }
}

// ------------------------------------------------------------------ the dense bias and its gradient
// out[h][i][j] = table[map[clamp(j - i - q_start)]][h]: bound by the stores.  A workgroup writes 16-byte chunks of one head's flat [Sq Sk]
// block (aligned in memory, whatever Sk is); a chunk whose distances all lie beyond the map's changes is one value.
template <class T>
__global__ void __launch_bounds__(256) la_bias_dense(const void* table, const int32_t* map, int H, int nb, int maxd, int Sq, int Sk, int q_start,
                                                     int chunks_per_wg, void* out) {
    constexpr int EPC = T::EPC;
    extern __shared__ float val[];  // [2 maxd + 1]
    const int head = blockIdx.y, tid = threadIdx.x, nd = 2 * maxd + 1;
    for (int x = tid; x < nd; x += 256) {
        const int t = map[x];
        val[x] = t >= 0 && t < nb ? T::elem(table, (int64_t)t * H + head) : __builtin_nanf("");
    }
    __syncthreads();
    const int64_t n = (int64_t)Sq * Sk, base = head * n;
    const int skew = (int)(base % EPC);
    const int64_t chunks = (n + skew + EPC - 1) / EPC;
    int64_t c = (int64_t)blockIdx.x * chunks_per_wg + tid;
    const int64_t cend = min(chunks, ((int64_t)blockIdx.x + 1) * chunks_per_wg);
    if (c >= cend) return;
    // row and column of the chunk's first element (the head's first chunk may begin before it: f < 0), then stepped by 256 chunks
    int64_t f = c * EPC - skew;
    int i = (int)(max(f, (int64_t)0) / Sk), j = (int)(f - (int64_t)i * Sk);
    const int di = 256 * EPC / Sk, dj = 256 * EPC - di * Sk;
    for (; c < cend; c += 256, f += 256 * EPC) {
        float v[EPC];
        const int d0 = j - i - q_start;
        if (f >= 0 && j + EPC <= Sk && (d0 + EPC - 1 <= -maxd || d0 >= maxd)) {
            const float x = val[d0 >= maxd ? nd - 1 : 0];
#pragma unroll
            for (int e = 0; e < EPC; ++e) v[e] = x;
        } else {
            int ii = i, jj = j;
#pragma unroll
            for (int e = 0; e < EPC; ++e) {
                v[e] = val[min(max(jj - ii - q_start, -maxd), maxd) + maxd];
                if (++jj == Sk) {
                    jj = 0;
                    ++ii;
                }
            }
        }
        if (f >= 0 && f + EPC <= n) {
            if constexpr (T::F32) {
                *reinterpret_cast<float4*>(static_cast<float*>(out) + base + f) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    q[k] = T::F16 ? (uint32_t)f16_bits(v[2 * k]) | (uint32_t)f16_bits(v[2 * k + 1]) << 16
                                  : (uint32_t)bf16_bits(v[2 * k]) | (uint32_t)bf16_bits(v[2 * k + 1]) << 16;
                *reinterpret_cast<uint4*>(static_cast<u16*>(out) + base + f) = make_uint4(q[0], q[1], q[2], q[3]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < EPC; ++e)
                if (f + e >= 0 && f + e < n) {
                    if constexpr (T::F32) static_cast<float*>(out)[base + f + e] = v[e];
                    else static_cast<u16*>(out)[base + f + e] = T::F16 ? f16_bits(v[e]) : bf16_bits(v[e]);
                }
        }
        i += di;
        j += dj;
        if (j >= Sk) {
            j -= Sk;
            ++i;
        }
    }
}

// Sums of a dense gradient [B][H][Sq][Sk] by distance: a workgroup takes `rows` rows of one (dialog, head).  The distances at which the map
// changes are summed along their diagonals, one thread each (neighbouring threads read neighbouring columns); what lies left and right of
// them goes, 16 bytes at a time, into two sums.  Bound by the one read of the gradient.
template <class T>
__global__ void __launch_bounds__(256) la_bias_grad(const void* dbias, LaParams p, int rows, int64_t total) {
    constexpr int EPC = T::EPC;
    extern __shared__ float sh[];  // 8 words for the range, 8 for the sums
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int lo, hi;
    bias_range(p, reinterpret_cast<int*>(sh), tid, lo, hi);
    const int64_t head = blockIdx.y;  // dialog and head
    const int i0 = blockIdx.x * rows, i1 = min(p.Sq, i0 + rows);
    const int64_t base = head * p.Sq * p.Sk;
    const int nd = 2 * p.maxd + 1;
    float* out = p.tpart + (head * gridDim.x + blockIdx.x) * (int64_t)(nd + 2);
    for (int x = tid; x < nd; x += 256) {
        const int d = x - p.maxd;
        float sum = 0.f;
        if (d >= lo && d <= hi) {
            const int a = max(i0, -d - p.q_start), z = min(i1, p.Sk - d - p.q_start);  // rows where 0 <= i + q_start + d < Sk
            for (int i = a; i < z; ++i) sum += T::elem(dbias, base + (int64_t)i * p.Sk + i + p.q_start + d);
        }
        out[x] = sum;
    }
    float left = 0.f, right = 0.f;
    for (int i = i0 + wave; i < i1; i += 4) {
        const int64_t row = base + (int64_t)i * p.Sk;
        const int jl = min(max(i + p.q_start + lo, 0), p.Sk), jr = min(max(i + p.q_start + hi + 1, 0), p.Sk);  // [0, jl) left, [jr, Sk) right
        const int64_t l_end = row + jl, r_beg = row + jr, end = row + p.Sk;
        for (int64_t c = row / EPC + lane; c * EPC < end; c += 64) {
            const int64_t f = c * EPC;
            if (f >= l_end && f + EPC <= r_beg) continue;
            float v[EPC];
            if (f + EPC <= total) {
                const void* at[2] = {dbias, nullptr};
                const uint4 x = T::load(at, f);
                if constexpr (T::F32) {
                    const float4 y = __builtin_bit_cast(float4, x);
                    v[0] = y.x;
                    v[1] = y.y;
                    v[2] = y.z;
                    v[3] = y.w;
                } else {
                    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        v[2 * k] = T::to_f32((u16)y[k]);
                        v[2 * k + 1] = T::to_f32((u16)(y[k] >> 16));
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < EPC; ++e) v[e] = f + e < total ? T::elem(dbias, f + e) : 0.f;
            }
            float sl = 0.f, sr = 0.f;
#pragma unroll
            for (int e = 0; e < EPC; ++e) {
                sl += f + e >= row && f + e < l_end ? v[e] : 0.f;
                sr += f + e >= r_beg && f + e < end ? v[e] : 0.f;
            }
            left += sl;
            right += sr;
        }
    }
    left = wave_sum(left);
    right = wave_sum(right);
    if (lane == 0) {
        sh[8 + wave] = left;
        sh[12 + wave] = right;
    }
    __syncthreads();
    if (tid == 0) {
        out[nd] = sh[8] + sh[9] + sh[10] + sh[11];
        out[nd + 1] = sh[12] + sh[13] + sh[14] + sh[15];
    }
}

// ------------------------------------------------------------------ host side
constexpr int MAX_DIST = 512, MAX_BUCKETS = 1024, MAX_SPLITS = 64;
constexpr int64_t TARGET_WGS = 512;  // two workgroups on each of 256 CUs

int pad_dim(int D) { return (D + 31) / 32 * 32; }

struct Plan {
    bool few;  // 32 rows a workgroup, the waves split the keys
    int nrt, ns;
    int nrt_q, ns_q, nrt_k, ns_k;
    size_t fwd_bytes, delta, part, tpart, bwd_bytes;
};

int pick_splits(int64_t base, int tiles) {
    if (base <= 0 || tiles <= 1) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({TARGET_WGS / base, (int64_t)tiles, (int64_t)MAX_SPLITS}));
}

Plan make_plan(const didi_long_attn_args* a) {
    Plan q{};
    const bool f32 = a->dtype == DIDI_DT_FP32 || a->Q_lo;
    const int G = a->heads / a->kv_heads;
    const int HG = a->table ? a->heads : a->kv_heads, Gr = a->table ? 1 : G;
    const int64_t R = (int64_t)Gr * a->Sq, rows = (int64_t)a->B * a->heads * a->Sq;
    q.few = R <= 32;
    q.nrt = (int)((R + (q.few ? 31 : 127)) / (q.few ? 32 : 128));
    q.ns = pick_splits((int64_t)a->B * HG * q.nrt, cdiv(a->Sk, q.few ? 128 : f32 ? 32 : 64));
    q.fwd_bytes = q.ns > 1 ? (size_t)q.ns * rows * (a->D + 2) * 4 : 0;
    q.nrt_q = (int)((R + 127) / 128);
    q.ns_q = pick_splits((int64_t)a->B * HG * q.nrt_q, cdiv(a->Sk, f32 ? 32 : 64));
    q.nrt_k = cdiv(a->Sk, 128);
    q.ns_k = pick_splits((int64_t)a->B * a->kv_heads * q.nrt_k, G * cdiv(a->Sq, f32 ? 32 : 64));
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    q.delta = up((size_t)2 * rows * 4);
    q.part = up(std::max(q.ns_q > 1 ? (size_t)q.ns_q * rows * a->D * 4 : 0, q.ns_k > 1 ? (size_t)2 * q.ns_k * a->B * a->kv_heads * a->Sk * a->D * 4 : 0));
    q.tpart = a->dtable ? up((size_t)a->B * a->heads * q.nrt_q * q.ns_q * (2 * a->max_distance + 3) * 4) : 0;
    q.bwd_bytes = q.delta + q.part + q.tpart;
    return q;
}

bool lds_opt_in(const void* fn, size_t bytes) {
    static std::mutex mu;
    if (bytes <= 64 * 1024) return true;
    std::lock_guard<std::mutex> lock(mu);
    return hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) == hipSuccess;
}

bool aligned(const void* p, int64_t batch, int64_t ld, int bytes, int elem) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && batch * elem % bytes == 0 && ld * elem % bytes == 0;
}

int check_args(const didi_long_attn_args* a, bool bwd) {
    DIDI_CHECK_ARG(a && a->B >= 0 && a->Sq >= 0 && a->Sk >= 0 && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->D > 0);
    DIDI_CHECK_ARG(a->dtype == DIDI_DT_BF16 || a->dtype == DIDI_DT_FP16 || a->dtype == DIDI_DT_FP32);
    DIDI_CHECK_ARG(a->scale >= 0.f && a->scale < INFINITY && a->drop_p >= 0.f && a->drop_p < 1.f && a->q_start >= 0);
    const bool planes = a->Q_lo || a->K_lo || a->V_lo, f32 = a->dtype == DIDI_DT_FP32;
    if (planes) DIDI_CHECK_ARG(!f32 && (a->Q_lo || !a->Q) && (a->K_lo || !a->K) && (a->V_lo || !a->V) && !bwd && !a->table);
    DIDI_CHECK_ARG(!(f32 && a->O_lo));
    if (a->D > 128 || a->D % (f32 || planes ? 4 : 8) != 0) return DIDI_ERR_UNSUPPORTED;
    if (a->table) {
        DIDI_CHECK_ARG(a->buckets && a->num_buckets > 0 && a->max_distance > 0);
        if (a->max_distance > MAX_DIST || a->num_buckets > MAX_BUCKETS) return DIDI_ERR_UNSUPPORTED;
    }
    DIDI_CHECK_ARG(a->table || !a->dtable);
    // sizes the kernels' 32-bit counts can hold: positions, packed rows, workgroups
    const int64_t lim = (int64_t)1 << 30;
    if ((int64_t)a->Sq * a->heads > lim || a->Sk > lim || (int64_t)a->q_start + a->Sq > lim || (int64_t)a->B * a->heads > (1 << 20)) return DIDI_ERR_UNSUPPORTED;
    const int64_t wq = (int64_t)a->heads * a->D, wk = (int64_t)a->kv_heads * a->D;
    const int e = f32 ? 4 : 2, al = planes ? 8 : 16;
    struct Op {
        const void* p;
        int64_t batch;
        int ld, S;
        int64_t w;
        bool need, written;
    } ops[] = {
        {a->Q, a->q_batch, a->ldq, a->Sq, wq, true, false},   {a->K, a->k_batch, a->ldk, a->Sk, wk, true, false},
        {a->V, a->v_batch, a->ldv, a->Sk, wk, true, false},   {a->O, a->o_batch, a->ldo, a->Sq, wq, true, !bwd},
        {a->Q_lo, a->q_batch, a->ldq, a->Sq, wq, false, false}, {a->K_lo, a->k_batch, a->ldk, a->Sk, wk, false, false},
        {a->V_lo, a->v_batch, a->ldv, a->Sk, wk, false, false}, {a->O_lo, a->o_batch, a->ldo, a->Sq, wq, false, !bwd},
        {a->dO, a->do_batch, a->lddo, a->Sq, wq, bwd, false}, {a->dQ, a->dq_batch, a->lddq, a->Sq, wq, bwd, true},
        {a->dK, a->dk_batch, a->lddk, a->Sk, wk, bwd, true},  {a->dV, a->dv_batch, a->lddv, a->Sk, wk, bwd, true},
    };
    for (const Op& o : ops) {
        if (a->B == 0 || o.S == 0 || (!bwd && &o >= ops + 8)) continue;  // the forward does not look at the gradients' fields
        if (o.need) DIDI_CHECK_ARG(o.p);
        if (!o.p) continue;
        DIDI_CHECK_ARG(o.ld >= o.w || o.S == 1);
        DIDI_CHECK_ARG(o.batch >= 0 && aligned(o.p, o.batch, o.ld, al, e));
        if (o.written && a->B > 1) DIDI_CHECK_ARG(o.batch >= (int64_t)(o.S - 1) * o.ld + o.w);  // dialogs of an output may not overlap
    }
    DIDI_CHECK_ARG(!bwd || a->lse || a->B == 0 || a->Sq == 0);
    return DIDI_OK;
}

LaParams make_params(const didi_long_attn_args* a) {
    LaParams p{};
    p.B = a->B; p.H = a->heads; p.Hk = a->kv_heads; p.G = a->heads / a->kv_heads; p.Sq = a->Sq; p.Sk = a->Sk; p.D = a->D;
    p.HG = a->table ? a->heads : a->kv_heads;
    p.Gr = a->table ? 1 : p.G;
    p.causal = a->causal != 0; p.q_start = a->q_start;
    p.scale = a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)a->D);
    p.sc = p.scale * LOG2E;
    p.mask = a->key_mask; p.count = a->key_count;
    p.Q[0] = a->Q; p.Q[1] = a->Q_lo; p.K[0] = a->K; p.K[1] = a->K_lo; p.V[0] = a->V; p.V[1] = a->V_lo;
    p.dO = a->dO; p.O[0] = a->O; p.O[1] = a->O_lo; p.Ow[0] = a->O; p.Ow[1] = a->O_lo;
    p.dQ = a->dQ; p.dK = a->dK; p.dV = a->dV;
    p.qb = a->q_batch; p.kb = a->k_batch; p.vb = a->v_batch; p.ob = a->o_batch; p.dob = a->do_batch;
    p.dqb = a->dq_batch; p.dkb = a->dk_batch; p.dvb = a->dv_batch;
    p.ldq = a->ldq; p.ldk = a->ldk; p.ldv = a->ldv; p.ldo = a->ldo; p.lddo = a->lddo; p.lddq = a->lddq; p.lddk = a->lddk; p.lddv = a->lddv;
    p.lse = a->lse;
    p.table = a->table; p.map = a->buckets; p.nb = a->num_buckets; p.maxd = a->table ? a->max_distance : 0;
    p.drop_p = a->drop_p;
    p.inv_keep = a->drop_p > 0.f ? 1.0f / (1.0f - a->drop_p) : 1.f;
    p.thr = (uint32_t)fminf(a->drop_p * 4294967296.0f, 4294967040.0f);
    p.seed = a->seed; p.offset = a->offset;
    return p;
}

template <class T, int DP, int WK>
int run_forward(const LaParams& p, hipStream_t st) {
    using C = FwdCfg<T, DP, WK>;
    const size_t lds = C::LDS + (p.table ? (size_t)(2 * p.maxd + 1 + 2 * PADB + 8) * 4 : 0);
    if (!lds_opt_in(reinterpret_cast<const void*>(&la_forward<T, DP, WK>), lds)) return DIDI_ERR_LAUNCH;
    la_forward<T, DP, WK><<<(unsigned)((int64_t)p.B * p.HG * p.nrt * p.ns), 256, lds, st>>>(p);
    DIDI_LAUNCH_CHECK();
    if (p.ns > 1) {
        la_join<T><<<(unsigned)(((int64_t)p.B * p.H * p.Sq * (p.D / 4) + 255) / 256), 256, 0, st>>>(p);
        DIDI_LAUNCH_CHECK();
    }
    return DIDI_OK;
}
template <class T, int DP>
int run_forward_dp(const LaParams& p, bool few, hipStream_t st) {
    return few ? run_forward<T, DP, 4>(p, st) : run_forward<T, DP, 1>(p, st);
}
template <class T>
int run_forward_t(const LaParams& p, bool few, hipStream_t st) {
    switch (pad_dim(p.D)) {
        case 32: return run_forward_dp<T, 32>(p, few, st);
        case 64: return run_forward_dp<T, 64>(p, few, st);
        case 96: return run_forward_dp<T, 96>(p, few, st);
        default: return run_forward_dp<T, 128>(p, few, st);
    }
}

template <class T, int DP>
int run_backward(LaParams p, const Plan& q, void* dtable, hipStream_t st) {
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    float* part = p.part;
    if (rows > 0) {
        using C = BwdQCfg<T, DP>;
        p.nrt = q.nrt_q;
        p.ns = q.ns_q;
        const size_t len = 2 * p.maxd + 1 + 2 * PADB, lds = C::LDS + (p.table ? (len * 9 + 8) * 4 : 0);
        if (!lds_opt_in(reinterpret_cast<const void*>(&la_backward_q<T, DP>), lds)) return DIDI_ERR_LAUNCH;
        la_backward_q<T, DP><<<(unsigned)((int64_t)p.B * p.HG * p.nrt * p.ns), 256, lds, st>>>(p);
        DIDI_LAUNCH_CHECK();
        if (p.ns > 1) {
            la_sum_parts<T><<<(unsigned)((rows * (p.D / 4) + 255) / 256), 256, 0, st>>>(part, p.ns, rows, p.Sq, p.H, p.D, p.dQ, p.dqb, p.lddq);
            DIDI_LAUNCH_CHECK();
        }
    }
    if (dtable) {
        la_table_sum<T><<<p.H, 1024, (size_t)4 * (2 * p.maxd + 3) * 4, st>>>(p.tpart, p.map, rows > 0 ? p.B : 0, p.H, q.nrt_q * q.ns_q, p.nb, p.maxd, dtable);
        DIDI_LAUNCH_CHECK();
    }
    const int64_t krows = (int64_t)p.B * p.Hk * p.Sk;
    if (krows > 0) {
        using C = BwdKCfg<T, DP>;
        p.nrt = q.nrt_k;
        p.ns = q.ns_k;
        p.part2 = part + (int64_t)p.ns * krows * p.D;
        const size_t lds = C::LDS + (p.table ? (size_t)(2 * p.maxd + 1 + 2 * PADB + 8) * 4 : 0);
        if (!lds_opt_in(reinterpret_cast<const void*>(&la_backward_kv<T, DP>), lds)) return DIDI_ERR_LAUNCH;
        la_backward_kv<T, DP><<<(unsigned)((int64_t)p.B * p.Hk * p.nrt * p.ns), 256, lds, st>>>(p);
        DIDI_LAUNCH_CHECK();
        if (p.ns > 1) {
            const unsigned grid = (unsigned)((krows * (p.D / 4) + 255) / 256);
            la_sum_parts<T><<<grid, 256, 0, st>>>(part, p.ns, krows, p.Sk, p.Hk, p.D, p.dK, p.dkb, p.lddk);
            la_sum_parts<T><<<grid, 256, 0, st>>>(p.part2, p.ns, krows, p.Sk, p.Hk, p.D, p.dV, p.dvb, p.lddv);
            DIDI_LAUNCH_CHECK();
        }
    }
    return DIDI_OK;
}
template <class T>
int run_backward_t(const LaParams& p, const Plan& q, void* dtable, hipStream_t st) {
    switch (pad_dim(p.D)) {
        case 32: return run_backward<T, 32>(p, q, dtable, st);
        case 64: return run_backward<T, 64>(p, q, dtable, st);
        case 96: return run_backward<T, 96>(p, q, dtable, st);
        default: return run_backward<T, 128>(p, q, dtable, st);
    }
}

}  // namespace

extern "C" size_t didi_long_attention_workspace_bytes(const didi_long_attn_args* a, int backward) {
    if (check_args(a, backward != 0) != DIDI_OK) return 0;
    const Plan q = make_plan(a);
    return backward ? q.bwd_bytes : q.fwd_bytes;
}

extern "C" int didi_long_attention_forward(const didi_long_attn_args* a, void* stream) {
    if (const int rc = check_args(a, false)) return rc;
    if (a->B == 0 || a->Sq == 0) return DIDI_OK;
    const Plan q = make_plan(a);
    if (q.fwd_bytes && (!a->workspace || a->workspace_bytes < q.fwd_bytes)) return DIDI_ERR_WORKSPACE;
    DIDI_CHECK_ARG((reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0);
    LaParams p = make_params(a);
    p.nrt = q.nrt;
    p.ns = q.ns;
    p.part = static_cast<float*>(a->workspace);
    p.ml = p.part + (int64_t)q.ns * a->B * a->heads * a->Sq * a->D;
    hipStream_t st = as_stream(stream);
    if (a->Q_lo) return a->dtype == DIDI_DT_FP16 ? run_forward_t<EPlanes<true>>(p, q.few, st) : run_forward_t<EPlanes<false>>(p, q.few, st);
    if (a->dtype == DIDI_DT_FP32) return run_forward_t<EF32>(p, q.few, st);
    return a->dtype == DIDI_DT_FP16 ? run_forward_t<E16<true>>(p, q.few, st) : run_forward_t<E16<false>>(p, q.few, st);
}

extern "C" int didi_long_attention_backward(const didi_long_attn_args* a, void* stream) {
    if (const int rc = check_args(a, true)) return rc;
    const Plan q = make_plan(a);
    if (q.bwd_bytes && (!a->workspace || a->workspace_bytes < q.bwd_bytes)) return DIDI_ERR_WORKSPACE;
    DIDI_CHECK_ARG((reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0);
    LaParams p = make_params(a);
    char* ws = static_cast<char*>(a->workspace);
    p.delta = reinterpret_cast<float*>(ws);
    p.part = reinterpret_cast<float*>(ws + q.delta);
    p.tpart = a->dtable ? reinterpret_cast<float*>(ws + q.delta + q.part) : nullptr;
    hipStream_t st = as_stream(stream);
    if (a->dtype == DIDI_DT_FP32) return run_backward_t<EF32>(p, q, a->dtable, st);
    return a->dtype == DIDI_DT_FP16 ? run_backward_t<E16<true>>(p, q, a->dtable, st) : run_backward_t<E16<false>>(p, q, a->dtable, st);
}

static int check_bias(const int32_t* buckets, int dtype, int heads, int num_buckets, int max_distance, int Sq, int Sk, int q_start) {
    DIDI_CHECK_ARG(buckets && heads > 0 && num_buckets > 0 && max_distance > 0 && Sq >= 0 && Sk >= 0 && q_start >= 0);
    DIDI_CHECK_ARG(dtype == DIDI_DT_BF16 || dtype == DIDI_DT_FP16 || dtype == DIDI_DT_FP32);
    const int64_t lim = (int64_t)1 << 30;
    if (max_distance > MAX_DIST || num_buckets > MAX_BUCKETS || heads > 65535 || Sk > lim || (int64_t)q_start + Sq > lim) return DIDI_ERR_UNSUPPORTED;
    return DIDI_OK;
}

extern "C" int didi_relative_bias(const void* table, const int32_t* buckets, int dtype, int heads, int num_buckets, int max_distance, int Sq, int Sk,
                                  int q_start, void* out, void* stream) {
    if (const int rc = check_bias(buckets, dtype, heads, num_buckets, max_distance, Sq, Sk, q_start)) return rc;
    if (Sq == 0 || Sk == 0) return DIDI_OK;
    DIDI_CHECK_ARG(table && out && (reinterpret_cast<uintptr_t>(out) & 15) == 0);
    const int epc = dtype == DIDI_DT_FP32 ? 4 : 8;
    const int64_t chunks = ((int64_t)Sq * Sk + 2 * epc - 1) / epc;
    // enough workgroups to fill the card, at most 16 chunks per thread
    const int per = 256 * (int)std::max<int64_t>(1, std::min<int64_t>(16, chunks * heads / (256 * 2048)));
    const dim3 grid((unsigned)((chunks + per - 1) / per), heads);
    const size_t lds = (size_t)(2 * max_distance + 1) * 4;
    hipStream_t st = as_stream(stream);
#define DIDI_BIAS(T) la_bias_dense<T><<<grid, 256, lds, st>>>(table, buckets, heads, num_buckets, max_distance, Sq, Sk, q_start, per, out)
    if (dtype == DIDI_DT_FP32) DIDI_BIAS(EF32);
    else if (dtype == DIDI_DT_FP16) DIDI_BIAS(E16<true>);
    else DIDI_BIAS(E16<false>);
#undef DIDI_BIAS
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}

// rows of the gradient one workgroup takes: 64, fewer where that would leave the card empty
static int grad_rows(int64_t bh, int Sq) { return (int)std::max<int64_t>(4, std::min<int64_t>(64, bh * Sq / 2048)); }

extern "C" size_t didi_relative_bias_backward_bytes(int B, int heads, int max_distance, int Sq) {
    if (B <= 0 || heads <= 0 || Sq <= 0 || max_distance <= 0 || max_distance > MAX_DIST) return 0;
    return (size_t)B * heads * cdiv(Sq, grad_rows((int64_t)B * heads, Sq)) * (2 * max_distance + 3) * 4;
}

extern "C" int didi_relative_bias_backward(const void* dbias, const int32_t* buckets, int dtype, int B, int heads, int num_buckets, int max_distance,
                                           int Sq, int Sk, int q_start, void* dtable, void* workspace, void* stream) {
    if (const int rc = check_bias(buckets, dtype, heads, num_buckets, max_distance, Sq, Sk, q_start)) return rc;
    DIDI_CHECK_ARG(B >= 0 && dtable);
    const bool any = B > 0 && Sq > 0 && Sk > 0;
    if ((int64_t)B * heads > 65535) return DIDI_ERR_UNSUPPORTED;
    hipStream_t st = as_stream(stream);
    LaParams p{};
    p.Sq = Sq; p.Sk = Sk; p.q_start = q_start; p.map = buckets; p.nb = num_buckets; p.maxd = max_distance;
    p.tpart = static_cast<float*>(workspace);
    int parts = 0;
    if (any) {
        DIDI_CHECK_ARG(dbias && workspace && (reinterpret_cast<uintptr_t>(dbias) & 15) == 0);
        const int rows = grad_rows((int64_t)B * heads, Sq);
        parts = cdiv(Sq, rows);
        const dim3 grid(parts, B * heads);
        const int64_t total = (int64_t)B * heads * Sq * Sk;
#define DIDI_GRAD(T) la_bias_grad<T><<<grid, 256, 16 * 4, st>>>(dbias, p, rows, total)
        if (dtype == DIDI_DT_FP32) DIDI_GRAD(EF32);
        else if (dtype == DIDI_DT_FP16) DIDI_GRAD(E16<true>);
        else DIDI_GRAD(E16<false>);
#undef DIDI_GRAD
        DIDI_LAUNCH_CHECK();
    }
    const size_t lds = (size_t)4 * (2 * max_distance + 3) * 4;
#define DIDI_SUM(T) la_table_sum<T><<<heads, 1024, lds, st>>>(p.tpart, buckets, any ? B : 0, heads, std::max(parts, 1), num_buckets, max_distance, dtable)
    if (dtype == DIDI_DT_FP32) DIDI_SUM(EF32);
    else if (dtype == DIDI_DT_FP16) DIDI_SUM(E16<true>);
    else DIDI_SUM(E16<false>);
#undef DIDI_SUM
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}
