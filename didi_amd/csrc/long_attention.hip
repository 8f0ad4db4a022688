// Host side of the attention of any lengths -- argument checks, how launches are cut, workspaces, the C entries -- and the dense relative
// position bias with its gradient.  The mathematics and the kernels: long_attention.hpp.
#include <numeric>
#include <utility>

#include "long_attention.hpp"

using namespace la;

namespace {

// ------------------------------------------------------------------ the dense bias and its gradient
// out[h][i][j] = table[map[clamp(j - i - q_start)]][h]: bound by the stores.  A workgroup writes 16-byte chunks of one head's flat [Sq Sk]
// block (aligned in memory, whatever Sk is); a chunk whose distances all lie beyond the map's changes is one value.  32 heads of 2048 x 2047
// bf16: 52 us, 5.2 TB/s.
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
    // row and column of the chunk's first element, then stepped by 256 chunks.  The head's first chunk may begin before it: its row is then
    // negative and its column the one that the steps go on from (0 <= j < Sk always)
    int64_t f = c * EPC - skew;
    int i = f >= 0 ? (int)(f / Sk) : -(int)((skew + (int64_t)Sk - 1) / Sk), j = (int)(f - (int64_t)i * Sk);
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

// Sums of a dense gradient [B][H][Sq][Sk] by distance: a workgroup takes `rows` rows of one (dialog, head).  The distances at which the map
// changes are summed along their diagonals, one thread each (neighbouring threads read neighbouring columns); what lies left and right of
// them goes, 16 bytes at a time, into two sums.  Bound by the one read of the gradient: 32 heads of 2048 x 2047 bf16 86 us, 3.1 TB/s (the
// diagonals are read two bytes a lane), and 9 us for the table's sums.
template <class T>
__global__ void __launch_bounds__(256) la_bias_grad(const void* dbias, LaParams p, int rows) {
    constexpr int EPC = T::EPC;
    extern __shared__ float sh[];  // 8 words for the range, 8 for the sums
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int lo, hi;
    bias_range(p, reinterpret_cast<int*>(sh), tid, lo, hi);
    const int64_t head = blockIdx.y;  // dialog and head
    const int i0 = blockIdx.x * rows, i1 = min(p.Sq, i0 + rows);
    const int64_t base = head * p.Sq * p.Sk;
    const int nd = 2 * p.maxd + 1;
    const int b = (int)(blockIdx.y / (unsigned)p.H), h = (int)blockIdx.y - b * p.H;
    float* out = p.tpart + (((int64_t)h * p.B + b) * gridDim.x + blockIdx.x) * (nd + 2);
    for (int x = tid; x < nd; x += 256) {
        const int d = x - p.maxd;
        float sum = 0.f;
        if (d >= lo && d <= hi) {
            const int a = max(i0, -d - p.q_start), z = min(i1, p.Sk - d - p.q_start);  // rows where 0 <= i + q_start + d < Sk
#pragma unroll 16
            for (int i = a; i < z; ++i) sum += T::elem(dbias, base + (int64_t)i * p.Sk + i + p.q_start + d);
        }
        out[x] = sum;
    }
    // Two rows of a wave at a time, four 16-byte loads of each on their way.  A row's left part is cut from its first column on, its right part from
    // jr on, wherever that lies in memory (the loads need no alignment); what is left over at the ends of the two parts is read element by element.
    float left = 0.f, right = 0.f;
    const char* bytes = static_cast<const char*>(dbias);
    for (int ia = i0 + wave; ia < i1; ia += 8) {
        int64_t row[2];
        int jl[2], jr[2], nl[2], n[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int i = ia + 4 * r;
            row[r] = base + (int64_t)i * p.Sk;
            jl[r] = i < i1 ? min(max(i + p.q_start + lo, 0), p.Sk) : 0;
            jr[r] = i < i1 ? min(max(i + p.q_start + hi + 1, 0), p.Sk) : p.Sk;  // [0, jl) left, [jr, Sk) right
            nl[r] = jl[r] / EPC;
            n[r] = nl[r] + (p.Sk - jr[r]) / EPC;
        }
        for (int c0 = lane; c0 < max(n[0], n[1]); c0 += 256) {
            typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
            u4 x[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int c = c0 + 64 * u;
                    x[r][u] = u4{0, 0, 0, 0};
                    if (c < n[r]) x[r][u] = *reinterpret_cast<const u4*>(bytes + (row[r] + (c < nl[r] ? c * EPC : jr[r] + (c - nl[r]) * EPC)) * T::ES);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float v[EPC];
#pragma unroll
                    for (int e = 0; e < EPC; ++e) {
                        if constexpr (T::F32) v[e] = __builtin_bit_cast(float, (uint32_t)x[r][u][e]);
                        else v[e] = T::to_f32((u16)(x[r][u][e >> 1] >> (16 * (e & 1))));
                    }
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < EPC; e += 4) sum += (v[e] + v[e + 1]) + (v[e + 2] + v[e + 3]);
                    const bool is_left = c0 + 64 * u < nl[r];
                    left += is_left ? sum : 0.f;
                    right += is_left ? 0.f : sum;
                }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int tl = jl[r] % EPC, tr = (p.Sk - jr[r]) % EPC;
            if (lane < tl) left += T::elem(dbias, row[r] + jl[r] - 1 - lane);
            if (lane < tr) right += T::elem(dbias, row[r] + p.Sk - 1 - lane);
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

// The same for few elements of one dialog, in one launch: a workgroup takes a head, a thread a whole diagonal, then a wave a bucket.  Latency is all
// there is to it: a thread walks min(Sq, Sk) elements, sixteen at a time (12 heads: 64 x 64 fp32 6.5 us, bf16 9.1, the two launches 8.6 and a
// launch more for the host; 128 x 128 fp32 10.2 against 12.8 us, bf16 16.6 against 12.9; 64 x 900 bf16 22 against 12).
template <class T>
__global__ void __launch_bounds__(512) la_bias_grad_small(const void* dbias, const int32_t* map, int H, int nb, int maxd, int Sq, int Sk,
                                                          int q_start, void* out) {
    extern __shared__ float sums[];  // [Sq + Sk - 1], then their buckets
    const int h = blockIdx.x, n = Sq + Sk - 1, tid = threadIdx.x, lane = tid & 63;
    int* bucket = reinterpret_cast<int*>(sums + n);
    for (int x = tid; x < n; x += 512) {
        const int off = x - (Sq - 1);  // key - row
        const int a = max(0, -off), z = min(Sq, Sk - off);
        float sum = 0.f;
        const int64_t base = (int64_t)h * Sq * Sk + off;
#pragma unroll 16
        for (int i = a; i < z; ++i) sum += T::elem(dbias, base + (int64_t)i * (Sk + 1));
        sums[x] = sum;
        bucket[x] = map[min(max(off - q_start, -maxd), maxd) + maxd];
    }
    __syncthreads();
    for (int t = tid >> 6; t < nb; t += 8) {
        float sum = 0.f;
        for (int x = lane; x < n; x += 64) sum += bucket[x] == t ? sums[x] : 0.f;
        sum = wave_sum(sum);
        if (lane == 0) {
            if constexpr (T::F32) static_cast<float*>(out)[(int64_t)t * H + h] = sum;
            else static_cast<u16*>(out)[(int64_t)t * H + h] = T::F16 ? f16_bits(sum) : bf16_bits(sum);
        }
    }
}

// ------------------------------------------------------------------ host side
constexpr int MAX_DIST = 512, MAX_BUCKETS = 1024, MAX_SPLITS = 64;


// groups: row groups (dialogs x heads); rows of each; n: length of the contraction; one: its tile at wk = 1 (32 wk otherwise); most: the largest wk.
// wk = 1 from `full` workgroups on, 2 from `half` on, else 4 (us, 12 heads of 64 unless said): forward, 512 x 512 with a bias: 384 workgroups 20.3
// (wk = 2: 18.4), 768: 25.9 (32.9); 16 heads of 128, 1024 x 1024: 128 workgroups 37.8, wk = 2 28.8, 4: 39.2; 63 x 512, 48 pairs: wk = 2 11.1,
// 4 7.8.  More than one workgroup per block of rows costs a second launch and the partial sums' traffic: only where fewer than `target` would run,
// and at least four tiles each (33000 keys, 12 pairs, one token: 199 us unsplit, 24 with 32 to 42; 512 keys, 12 pairs: 9.7 unsplit, 11.0 with 2).
Cut cut(int64_t groups, int64_t rows, int64_t n, int one, int most, int64_t full, int64_t half, int64_t target) {
    Cut c{};
    c.wk = rows <= 32 || groups * cdiv(rows, 64) < half ? 4 : groups * cdiv(rows, 128) < full ? 2 : 1;
    c.wk = std::min(c.wk, most);
    c.nrt = cdiv(rows, 128 / c.wk);
    const int64_t base = std::max<int64_t>(1, groups * c.nrt), tile = c.wk == 1 ? one : 32 * c.wk, tiles = std::max<int64_t>(1, (n + tile - 1) / tile);
    c.ns = (int)std::max<int64_t>(1, std::min<int64_t>({target / base, tiles / 4, (int64_t)MAX_SPLITS}));
    c.per = (int)((tiles + c.ns - 1) / c.ns);
    return c;
}

Plan make_plan(const didi_long_attn_args* a) {
    Plan z{};
    const bool f32 = a->dtype == DIDI_DT_FP32;
    const int G = a->heads / a->kv_heads, one = f32 ? 32 : 64, most = max_share(f32, pad_dim(a->D));
    const int64_t HG = a->table ? a->heads : a->kv_heads, R = (int64_t)(a->table ? 1 : G) * a->Sq, rows = (int64_t)a->B * a->heads * a->Sq;
    // one token per row group: the keys are all there is to read, and dialogs of different lengths want smaller pieces (32 dialogs to 4096 keys:
    // 50.5 us unsplit, 45.6 to 47.4 with 2 to 4)
    const bool few = R <= 32;
    z.f = cut(a->B * HG, R, a->Sk, one, most, 512, 192, !few ? 256 : a->B * HG > 256 ? 1152 : 512);
    int most_q = most;  // wide biases: the sums by distance take the room of shared tiles
    if (a->table)
        while (most_q > 1 && 2 * stages(image_bytes(f32, pad_dim(a->D), most_q)) * image_bytes(f32, pad_dim(a->D), most_q) + sums_lds(a->max_distance) > MAX_LDS) most_q /= 2;
    z.q = cut(a->B * HG, R, a->Sk, one, most_q, 256, 192, 256);
    z.k = cut((int64_t)a->B * a->kv_heads, a->Sk, (int64_t)G * a->Sq, one, most, 128, 128, 128);  // 15 x 777 keys of 80: wk = 1 41.8 us, 2 40.5, 4 46.8 (of the whole backward)
    {  // the contraction of la_backward_kv is counted in tiles of each head
        const int64_t tile = z.k.wk == 1 ? one : 32 * z.k.wk, tiles = std::max<int64_t>(1, G * ((a->Sq + tile - 1) / tile));
        z.k.per = (int)((tiles + z.k.ns - 1) / z.k.ns);
    }
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    z.fwd_bytes = z.f.ns > 1 ? (size_t)z.f.ns * rows * (a->D + 2) * 4 : 0;
    z.rows = up((size_t)3 * rows * 4);
    z.part = up(std::max(z.q.ns > 1 ? (size_t)z.q.ns * rows * a->D * 4 : 0, z.k.ns > 1 ? (size_t)2 * z.k.ns * a->B * a->kv_heads * a->Sk * a->D * 4 : 0));
    z.tpart = a->dtable ? up((size_t)a->B * a->heads * z.q.nrt * z.q.ns * (2 * a->max_distance + 3) * 4) : 0;
    z.bwd_bytes = z.rows + z.part + z.tpart;
    return z;
}

bool aligned(const void* p, int64_t batch, int64_t ld, int bytes, int elem) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && batch * elem % bytes == 0 && ld * elem % bytes == 0;
}

int check_args(const didi_long_attn_args* a, bool bwd) {
    DIDI_CHECK_ARG(a && a->B >= 0 && a->Sq >= 0 && a->Sk >= 0 && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->D > 0);
    DIDI_CHECK_ARG(a->dtype == DIDI_DT_BF16 || a->dtype == DIDI_DT_FP16 || a->dtype == DIDI_DT_FP32);
    DIDI_CHECK_ARG((a->scale == 0.f || (a->scale >= 0x1p-126f && a->scale <= 0x1p127f)) && a->drop_p >= 0.f && a->drop_p < 1.f && a->q_start >= 0);
    const bool f32 = a->dtype == DIDI_DT_FP32;
    DIDI_CHECK_ARG(!(f32 && a->O_lo));
    if (a->D > 128 || a->D % (f32 ? 4 : 8) != 0) return DIDI_ERR_UNSUPPORTED;
    if (a->table) {
        DIDI_CHECK_ARG(a->buckets && a->num_buckets > 0 && a->max_distance > 0);
        if (a->max_distance > MAX_DIST || a->num_buckets > MAX_BUCKETS) return DIDI_ERR_UNSUPPORTED;
    }
    DIDI_CHECK_ARG(a->table || !a->dtable);
    // sizes the kernels' 32-bit counts can hold: positions, packed rows, workgroups
    const int64_t lim = (int64_t)1 << 30;
    for (int ld : {a->ldq, a->ldk, a->ldv, a->lddo})  // a tile of up to 128 rows lies within 2 GiB
        if (ld > (1 << 21)) return DIDI_ERR_UNSUPPORTED;
    if ((int64_t)a->heads * a->D > (1 << 21)) return DIDI_ERR_UNSUPPORTED;
    if ((int64_t)a->Sq * a->heads > lim || cdiv((int64_t)a->Sq * a->heads, 32) > 65535 || cdiv(a->Sk, 32) > 65535 || a->Sk > lim || (int64_t)a->q_start + a->Sq > lim || (int64_t)a->B * a->heads > (1 << 20)) return DIDI_ERR_UNSUPPORTED;
    const int64_t wq = (int64_t)a->heads * a->D, wk = (int64_t)a->kv_heads * a->D;
    const int e = f32 ? 4 : 2;
    struct Op {
        const void* p;
        int64_t batch;
        int ld, S;
        int64_t w;
        bool need, written;
    } ops[] = {
        {a->Q, a->q_batch, a->ldq, a->Sq, wq, true, false},   {a->K, a->k_batch, a->ldk, a->Sk, wk, true, false},
        {a->V, a->v_batch, a->ldv, a->Sk, wk, true, false},   {a->O, a->o_batch, a->ldo, a->Sq, wq, true, !bwd},
        {a->O_lo, a->o_batch, a->ldo, a->Sq, wq, false, !bwd},
        {a->dO, a->do_batch, a->lddo, a->Sq, wq, bwd, false}, {a->dQ, a->dq_batch, a->lddq, a->Sq, wq, bwd, true},
        {a->dK, a->dk_batch, a->lddk, a->Sk, wk, bwd, true},  {a->dV, a->dv_batch, a->lddv, a->Sk, wk, bwd, true},
    };
    for (const Op& o : ops) {
        if (a->B == 0 || o.S == 0 || (!bwd && &o >= ops + 5)) continue;  // the forward does not look at the gradients' fields
        if (o.need) DIDI_CHECK_ARG(o.p);
        if (!o.p) continue;
        DIDI_CHECK_ARG(o.ld >= o.w || o.S == 1);
        DIDI_CHECK_ARG(o.batch >= 0 && aligned(o.p, o.batch, o.ld, 16, e));
        // dialogs of an output may not overlap: one behind the other, or row by row in turn
        if (o.written && a->B > 1) DIDI_CHECK_ARG(o.batch >= (int64_t)(o.S - 1) * o.ld + o.w || (o.batch >= o.w && o.ld >= (int64_t)(a->B - 1) * o.batch + o.w));
    }
    DIDI_CHECK_ARG(!bwd || a->lse || a->B == 0 || a->Sq == 0);
    return DIDI_OK;
}

// An array of B dialogs of S rows in bytes; a contiguous one is a single row
struct Span {
    uintptr_t at;
    int64_t n[2], step[2], w;  // outer and inner count and stride
    Span(const void* p, int64_t B, int64_t batch, int64_t S, int64_t ld, int64_t width, int elem) : at(reinterpret_cast<uintptr_t>(p)), w(width * elem) {
        n[0] = B; step[0] = batch * elem;
        n[1] = S; step[1] = ld * elem;
        if (!p || B == 0 || S == 0 || width == 0) n[0] = 0;
        for (int k = 0; k < 2; ++k)
            if (n[k] == 1) step[k] = 0;  // an only row's or dialog's stride does not count
        if (n[0] > 1 && step[0] < step[1]) *this = turned();
    }
    Span turned() const {
        Span s = *this;
        std::swap(s.n[0], s.n[1]);
        std::swap(s.step[0], s.step[1]);
        return s;
    }
    Span(const void* p, int64_t bytes) : Span(p, 1, 0, 1, 0, bytes, 1) {}
    bool empty() const { return n[0] == 0 || n[1] == 0; }
    int64_t inner() const { return (n[1] - 1) * step[1] + w; }  // bytes from the first to behind the last of one outer step
    int64_t all() const { return (n[0] - 1) * step[0] + inner(); }
};

// whether [0, a) and [d, d + b) share nothing when both repeat every g
bool apart(int64_t d, int64_t a, int64_t b, int64_t g) {
    if (g == 0) return false;
    d = (d % g + g) % g;
    return d >= a && d + b <= g;
}

// Two arrays are apart within a common stride of all rows, or of the outer steps, or the outer strides are one and the outer steps that meet have rows
// that are
bool steps_apart(const Span& a, const Span& b) {
    const int64_t d = (int64_t)(b.at - a.at);
    const int64_t outer = std::gcd(a.step[0], b.step[0]), inner = std::gcd(a.step[1], b.step[1]);
    if (apart(d, a.w, b.w, std::gcd(outer, inner)) || apart(d, a.inner(), b.inner(), outer)) return true;
    const int64_t P = std::max(a.step[0], b.step[0]);
    if ((a.step[0] && a.step[0] != P) || (b.step[0] && b.step[0] != P) || P == 0 || a.inner() > P || b.inner() > P) return false;
    const int64_t r = (d % P + P) % P;  // an outer step of a meets the one of b that begins r behind it and the one that begins P - r before it
    for (const int64_t x : {r, r - P})
        if (x < a.inner() && -x < b.inner() && !apart(x, a.w, b.w, inner)) return false;
    return true;
}

// Whether two arrays share no element; false also where that cannot be shown.  An array of one row (dialog) a dialog (in all) is taken either way.
bool disjoint(const Span& a, const Span& b) {
    if (a.empty() || b.empty()) return true;
    const int64_t d = (int64_t)(b.at - a.at);
    if (d >= a.all() || -d >= b.all()) return true;
    const bool ta = a.n[0] == 1 || a.n[1] == 1, tb = b.n[0] == 1 || b.n[1] == 1;
    return steps_apart(a, b) || (ta && steps_apart(a.turned(), b)) || (tb && steps_apart(a, b.turned())) || (ta && tb && steps_apart(a.turned(), b.turned()));
}

// results over operands or over each other
int check_overlap(const didi_long_attn_args* a, bool bwd, size_t workspace) {
    const int e = a->dtype == DIDI_DT_FP32 ? 4 : 2;
    const int64_t wq = (int64_t)a->heads * a->D, wk = (int64_t)a->kv_heads * a->D;
    const int64_t table = a->table ? (int64_t)a->num_buckets * a->heads * e : 0;
    const Span O(a->O, a->B, a->o_batch, a->Sq, a->ldo, wq, e), lo(a->O_lo, a->B, a->o_batch, a->Sq, a->ldo, wq, e), lse(a->lse, (int64_t)a->B * a->heads * a->Sq * 4);
    const Span ws(a->workspace, (int64_t)workspace);
    const Span in[] = {Span(a->Q, a->B, a->q_batch, a->Sq, a->ldq, wq, e), Span(a->K, a->B, a->k_batch, a->Sk, a->ldk, wk, e),
                       Span(a->V, a->B, a->v_batch, a->Sk, a->ldv, wk, e), Span(a->key_mask, (int64_t)a->B * a->Sk * 4), Span(a->key_count, (int64_t)a->B * 4),
                       Span(a->table, table), Span(a->buckets, a->table ? (2 * (int64_t)a->max_distance + 1) * 4 : 0)};
    auto clear_of = [&](const Span& out) {
        for (const Span& s : in)
            if (!disjoint(out, s)) return false;
        return true;
    };
    if (!bwd) {
        const bool ok = clear_of(O) && clear_of(lo) && clear_of(lse) && clear_of(ws) && disjoint(O, lo) && disjoint(O, lse) && disjoint(O, ws) && disjoint(lo, lse) &&
                        disjoint(lo, ws) && disjoint(lse, ws);
        return ok ? DIDI_OK : DIDI_ERR_OVERLAP;
    }
    const Span out[] = {Span(a->dQ, a->B, a->dq_batch, a->Sq, a->lddq, wq, e), Span(a->dK, a->B, a->dk_batch, a->Sk, a->lddk, wk, e),
                        Span(a->dV, a->B, a->dv_batch, a->Sk, a->lddv, wk, e), Span(a->dtable, table), ws};
    const Span dO(a->dO, a->B, a->do_batch, a->Sq, a->lddo, wq, e);
    for (const Span& x : out) {
        if (!clear_of(x) || !disjoint(x, O) || !disjoint(x, lo) || !disjoint(x, lse) || !disjoint(x, dO)) return DIDI_ERR_OVERLAP;
        for (const Span* y = out; y != &x; ++y)
            if (!disjoint(x, *y)) return DIDI_ERR_OVERLAP;
    }
    return DIDI_OK;
}

LaParams make_params(const didi_long_attn_args* a, bool bwd) {
    LaParams p{};
    p.B = a->B; p.H = a->heads; p.Hk = a->kv_heads; p.G = a->heads / a->kv_heads; p.Sq = a->Sq; p.Sk = a->Sk; p.D = a->D;
    p.HG = a->table ? a->heads : a->kv_heads;
    p.Gr = a->table ? 1 : p.G;
    p.causal = a->causal != 0; p.q_start = a->q_start;
    p.scale = a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)a->D);
    p.sc = p.scale * LOG2E;
    p.mask = a->key_mask; p.count = a->key_count;
    p.Q = a->Q; p.K = a->K; p.V = a->V;
    p.dO = a->dO; p.O[0] = a->O; p.O[1] = a->O_lo; p.Ow[0] = a->O; p.Ow[1] = a->O_lo;
    p.dQ = a->dQ; p.dK = a->dK; p.dV = a->dV;
    p.qb = a->q_batch; p.kb = a->k_batch; p.vb = a->v_batch; p.ob = a->o_batch; p.dob = a->do_batch;
    p.dqb = a->dq_batch; p.dkb = a->dk_batch; p.dvb = a->dv_batch;
    // an only row's stride does not count, but the kernels' tiles are cut at rows x stride
    auto ld = [a](int stride, int S, int heads) { return S == 1 ? heads * a->D : stride; };
    p.ldq = ld(a->ldq, a->Sq, a->heads); p.ldo = ld(a->ldo, a->Sq, a->heads); p.lddo = ld(a->lddo, a->Sq, a->heads); p.lddq = ld(a->lddq, a->Sq, a->heads);
    p.ldk = ld(a->ldk, a->Sk, a->kv_heads); p.ldv = ld(a->ldv, a->Sk, a->kv_heads); p.lddk = ld(a->lddk, a->Sk, a->kv_heads); p.lddv = ld(a->lddv, a->Sk, a->kv_heads);
    p.lse = a->lse;
    p.table = a->table; p.map = a->buckets; p.nb = a->num_buckets; p.maxd = a->table ? a->max_distance : 0;
    p.thr = (uint32_t)fminf(a->drop_p * 4294967296.0f, 4294967040.0f);
    const float inv_keep = p.thr ? 1.0f / (1.0f - a->drop_p) : 1.f;
    p.on = std::min(inv_keep, bwd ? 32768.f : 128.f);
    p.rest = inv_keep / p.on;
    p.seed = a->seed; p.offset = a->offset;
    return p;
}

// what la_bias_grad_small takes (its comment has both sides)
bool grad_small(int B, int Sq, int Sk) { return B == 1 && std::min(Sq, Sk) <= 64 && (int64_t)Sq + Sk <= 512; }

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
    if (const int rc = check_overlap(a, false, q.fwd_bytes)) return rc;
    LaParams p = make_params(a, false);
    set_cut(p, q.f);
    p.part = static_cast<float*>(a->workspace);
    p.ml = p.part + (int64_t)q.f.ns * a->B * a->heads * a->Sq * a->D;
    hipStream_t st = as_stream(stream);
    if (a->dtype == DIDI_DT_FP32) return forward_fp32(p, q.f, st);
    return a->dtype == DIDI_DT_FP16 ? forward_fp16(p, q.f, st) : forward_bf16(p, q.f, st);
}

extern "C" int didi_long_attention_backward(const didi_long_attn_args* a, void* stream) {
    if (const int rc = check_args(a, true)) return rc;
    const Plan q = make_plan(a);
    if (q.bwd_bytes && (!a->workspace || a->workspace_bytes < q.bwd_bytes)) return DIDI_ERR_WORKSPACE;
    DIDI_CHECK_ARG((reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0);
    if (const int rc = check_overlap(a, true, q.bwd_bytes)) return rc;
    LaParams p = make_params(a, true);
    char* ws = static_cast<char*>(a->workspace);
    p.rows = reinterpret_cast<float*>(ws);
    p.part = reinterpret_cast<float*>(ws + q.rows);
    p.tpart = a->dtable ? reinterpret_cast<float*>(ws + q.rows + q.part) : nullptr;
    hipStream_t st = as_stream(stream);
    if (a->dtype == DIDI_DT_FP32) return backward_fp32(p, q, a->dtable, st);
    return a->dtype == DIDI_DT_FP16 ? backward_fp16(p, q, a->dtable, st) : backward_bf16(p, q, a->dtable, st);
}

static int check_bias(const int32_t* buckets, int dtype, int heads, int num_buckets, int max_distance, int Sq, int Sk, int q_start) {
    DIDI_CHECK_ARG(buckets && heads > 0 && num_buckets > 0 && max_distance > 0 && Sq >= 0 && Sk >= 0 && q_start >= 0);
    DIDI_CHECK_ARG(dtype == DIDI_DT_BF16 || dtype == DIDI_DT_FP16 || dtype == DIDI_DT_FP32);
    const int64_t lim = (int64_t)1 << 30;
    if (max_distance > MAX_DIST || num_buckets > MAX_BUCKETS || heads > 65535 || Sk > lim || (int64_t)q_start + Sq > lim) return DIDI_ERR_UNSUPPORTED;
    if ((int64_t)Sq * Sk > ((int64_t)1 << 40)) return DIDI_ERR_UNSUPPORTED;  // what the launch's grid holds, and more than any memory does
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

extern "C" size_t didi_relative_bias_backward_bytes(int B, int heads, int max_distance, int Sq, int Sk) {
    if (B <= 0 || heads <= 0 || Sq <= 0 || Sk <= 0 || max_distance <= 0 || max_distance > MAX_DIST || grad_small(B, Sq, Sk)) return 0;
    return (size_t)B * heads * cdiv(Sq, grad_rows((int64_t)B * heads, Sq)) * (2 * max_distance + 3) * 4;
}

extern "C" int didi_relative_bias_backward(const void* dbias, const int32_t* buckets, int dtype, int B, int heads, int num_buckets, int max_distance,
                                           int Sq, int Sk, int q_start, void* dtable, void* workspace, void* stream) {
    if (const int rc = check_bias(buckets, dtype, heads, num_buckets, max_distance, Sq, Sk, q_start)) return rc;
    DIDI_CHECK_ARG(B >= 0 && dtable);
    const bool any = B > 0 && Sq > 0 && Sk > 0;
    const int elem = dtype == DIDI_DT_FP32 ? 4 : 2;  // the loads need no more
    if ((int64_t)B * heads > 65535) return DIDI_ERR_UNSUPPORTED;
    hipStream_t st = as_stream(stream);
    LaParams p{};
    p.B = B; p.H = heads; p.Sq = Sq; p.Sk = Sk; p.q_start = q_start; p.map = buckets; p.nb = num_buckets; p.maxd = max_distance;
    p.tpart = static_cast<float*>(workspace);
    int parts = 0;
    if (any && grad_small(B, Sq, Sk)) {
        DIDI_CHECK_ARG(dbias && reinterpret_cast<uintptr_t>(dbias) % elem == 0);
#define DIDI_SMALL(T) la_bias_grad_small<T><<<heads, 512, (size_t)(Sq + Sk - 1) * 8, st>>>(dbias, buckets, heads, num_buckets, max_distance, Sq, Sk, q_start, dtable)
        if (dtype == DIDI_DT_FP32) DIDI_SMALL(EF32);
        else if (dtype == DIDI_DT_FP16) DIDI_SMALL(E16<true>);
        else DIDI_SMALL(E16<false>);
#undef DIDI_SMALL
        DIDI_LAUNCH_CHECK();
        return DIDI_OK;
    }
    if (any) {
        DIDI_CHECK_ARG(dbias && workspace && reinterpret_cast<uintptr_t>(dbias) % elem == 0);
        const int rows = grad_rows((int64_t)B * heads, Sq);
        parts = cdiv(Sq, rows);
        const dim3 grid(parts, B * heads);
#define DIDI_GRAD(T) la_bias_grad<T><<<grid, 256, 16 * 4, st>>>(dbias, p, rows)
        if (dtype == DIDI_DT_FP32) DIDI_GRAD(EF32);
        else if (dtype == DIDI_DT_FP16) DIDI_GRAD(E16<true>);
        else DIDI_GRAD(E16<false>);
#undef DIDI_GRAD
        DIDI_LAUNCH_CHECK();
    }
    const size_t lds = table_lds(max_distance, 1024);
#define DIDI_SUM(T) la_table_sum<T><<<heads, 1024, lds, st>>>(p.tpart, buckets, any ? B : 0, heads, std::max(parts, 1), num_buckets, max_distance, dtable)
    if (dtype == DIDI_DT_FP32) DIDI_SUM(EF32);
    else if (dtype == DIDI_DT_FP16) DIDI_SUM(E16<true>);
    else DIDI_SUM(E16<false>);
#undef DIDI_SUM
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}
