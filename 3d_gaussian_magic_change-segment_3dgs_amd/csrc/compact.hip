// compact.hip -- the compact-scene kernels of include/gsr_compact.h: 4-bit microscaled
// rows, colours from them with their gradients, eviction of the lightest Gaussians.
#include "gsr_internal.h"
#include "../../include/gsr_compact.h"

namespace gsr {
namespace {

constexpr int CP_THREADS = 256;

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(std::string("[gsr] ") + what + ": " + hipGetErrorString(e));
    return 0;
}

__host__ __device__ inline int mx_words(int K) { return (K + 7) / 8; }
__host__ __device__ inline int mx_blocks(int K) { return (K + GSR_MX_BLOCK - 1) / GSR_MX_BLOCK; }

// How the units of a row of a streamed tensor (R rows of `units`) go to blocks of `span`
// lanes: whole rows where a row fits, so that no lane divides (units 9 of a 768 span:
// 85 rows, 99.6 % of the lanes); pieces of a row otherwise.
struct Tiling {
    int units, rows;  // rows a block (0: pieces)
    uint32_t magic;   // 2^32 / units + 1: exact quotients of numbers below 2^32 / units
};
inline Tiling tiling(int units, int span) {
    return {units, units <= span ? span / units : 0, units > 1 ? (uint32_t)((1ULL << 32) / units + 1) : 0u};
}
inline long long tiling_blocks(const Tiling& t, long long R, int span) {
    return t.rows > 0 ? (R + t.rows - 1) / t.rows : (R * t.units + span - 1) / span;
}
template <int SPAN>
__device__ __forceinline__ bool tiling_place(const Tiling& t, uint32_t block, uint32_t local, long long R,
                                             long long& row, int& unit) {
    if (t.rows > 0) {
        const uint32_t r = t.units == 1 ? local : __umulhi(local, t.magic);
        row = (long long)block * t.rows + r;
        unit = (int)(local - r * t.units);
        return r < (uint32_t)t.rows && row < R;
    }
    const long long e = (long long)block * SPAN + local;
    row = e / t.units;
    unit = (int)(e - row * t.units);
    return row < R;
}

// ------------------------------------------------------------------ 4-bit rows --
// The gfx950 converts do the whole of the rounding: v_cvt_scalef32_pk_fp4_f32 divides by
// 2^(exponent field - 127) and rounds to E2M1 (nearest, ties to even, saturating; exponent
// field 0 is 2^-127, 255 is NaN when read back), so the scale byte goes in as the bits of a float.
typedef float f2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

typedef float v4a __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any word

__device__ __forceinline__ uint32_t mx_encode8(v4a lo, v4a hi, float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo.x, lo.y, scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo.z, lo.w, scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, hi.x, hi.y, scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, hi.z, hi.w, scale, 3);
    return w;
}

__device__ __forceinline__ void mx_decode8(uint32_t w, float scale, float* v) {
    const f2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    const f2v b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    const f2v c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
    const f2v d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// Scale byte of a block from the largest |x| as bits (an unsigned maximum: NaN and infinity
// come out on top).  floor(log2) - 2 is the exponent field less two, from 0 upwards.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e : 2u) - 2u;
}


// Values [k, k + 4) of a row of K (p: its value k), zeros behind its end.  A piece that ends with
// the row is read as the row's last four values, shifted: one load whatever the length.
__device__ __forceinline__ v4a load4(const float* p, int k, int K) {
    v4a r = {0.0f, 0.0f, 0.0f, 0.0f};
    if ((K & 3) == 0) {
        if (k < K) r = *reinterpret_cast<const v4a*>(p);
    } else if (K >= 4) {
        const int over = k + 4 - K;
        if (over < 4) {
            const v4a q = *reinterpret_cast<const v4a*>(over > 0 ? p - over : p);
            r.x = over <= 0 ? q.x : over == 1 ? q.y : over == 2 ? q.z : q.w;
            r.y = over <= 0 ? q.y : over == 1 ? q.z : over == 2 ? q.w : 0.0f;
            r.z = over <= 0 ? q.z : over == 1 ? q.w : 0.0f;
            r.w = over <= 0 ? q.w : 0.0f;
        }
    } else {
        if (k < K) r.x = p[0];
        if (k + 1 < K) r.y = p[1];
        if (k + 2 < K) r.z = p[2];
    }
    return r;
}
__device__ __forceinline__ uint32_t max_bits(uint32_t m, v4a v) {
    const uint32_t x = __float_as_uint(v.x) & 0x7FFFFFFFu, y = __float_as_uint(v.y) & 0x7FFFFFFFu,
                   z = __float_as_uint(v.z) & 0x7FFFFFFFu, w = __float_as_uint(v.w) & 0x7FFFFFFFu;
    const uint32_t a = x > y ? x : y, b = z > w ? z : w, c = a > b ? a : b;
    return m > c ? m : c;
}

// Four lanes per block, eight values (one code word) each; the four share the largest |x| through
// DPP.  A thread takes MXQ_PER such pieces, their loads in flight together.  Bound by memory: 1M rows of 45
// (206 MB, with the 12 bytes between them 218) 35 us, 6.2 TB/s.
constexpr int MXQ_PER = 2, MXQ_SPAN = CP_THREADS / 4 * MXQ_PER;
__global__ void __launch_bounds__(CP_THREADS) k_mx4_quantize(long long R, int K, Tiling t, const float* __restrict__ x,
                                                             long long stride, uint32_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
    const int nw = mx_words(K), sub = threadIdx.x & 3;
    v4a lo[MXQ_PER], hi[MXQ_PER];
    long long row[MXQ_PER];
    int b[MXQ_PER];
    bool in[MXQ_PER];  // the same for the four
#pragma unroll
    for (int u = 0; u < MXQ_PER; ++u) {
        in[u] = tiling_place<MXQ_SPAN>(t, blockIdx.x, u * (CP_THREADS / 4) + (threadIdx.x >> 2), R, row[u], b[u]);
        const int k0 = b[u] * GSR_MX_BLOCK + sub * 8;
        const float* p = x + row[u] * stride + k0;
        const int end = in[u] ? K : 0;
        lo[u] = load4(p, k0, end);
        hi[u] = load4(p + 4, k0 + 4, end);
    }
#pragma unroll
    for (int u = 0; u < MXQ_PER; ++u) {
        uint32_t m = max_bits(max_bits(0u, lo[u]), hi[u]);
        uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true);  // quad_perm 1 0 3 2
        m = m > o ? m : o;
        o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true);  // quad_perm 2 3 0 1
        m = m > o ? m : o;
        const uint32_t s = mx_scale_byte(m);
        const int w = b[u] * 4 + sub;
        if (in[u] && w < nw) codes[row[u] * nw + w] = s == 255u ? 0u : mx_encode8(lo[u], hi[u], mx_scale(s));
        if (in[u] && sub == 0) scales[row[u] * t.units + b[u]] = (uint8_t)s;
    }
}

// Four values (a half word of codes) per lane: a wave writes 1 KB in one piece, of rows as they lie.
// For the widths that the kernel below does not take.
__global__ void __launch_bounds__(CP_THREADS) k_mx4_dequantize(long long R, int K, Tiling t,
                                                               const uint16_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               float* __restrict__ x) {
    const int nb = mx_blocks(K), nh = 2 * mx_words(K);
    long long row;
    int h;
    if (!tiling_place<CP_THREADS>(t, blockIdx.x, threadIdx.x, R, row, h)) return;
    const uint32_t w = codes[row * nh + h];
    const float s = mx_scale(scales[row * nb + (h >> 3)]);
    const f2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
    const f2v b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    float* p = x + row * K + 4 * h;
    if (4 * h + 4 <= K) {
        *reinterpret_cast<v4a*>(p) = v4a{a.x, a.y, b.x, b.y};
    } else {
        const float v[3] = {a.x, a.y, b.x};
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (4 * h + j < K) p[j] = v[j];
    }
}

// The same by the output's flat index: a lane's four values are a whole 16-byte unit of it whatever K,
// so every cache line is written by one instruction and can pass by the caches (with 45 values a row,
// pieces that follow the rows leave parts of lines: 1M rows 33 us through the caches, whose lines then
// stand in the way of the next kernel's reads, and 57 past them).  The four lie in at most two rows (K >= 4) and
// under at most two scales, which are neighbours (K mod 32 not 1 or 2).  Quantise and back of 1M
// rows of 45, 88 -> 74 us; of 300k rows of 24, 15.9 -> 15.5; of 10k rows of 45, no change.
constexpr int MXD_SPAN = 4 * CP_THREADS;
inline bool mxd_flat(int K) { return K >= 4 && K % GSR_MX_BLOCK != 1 && K % GSR_MX_BLOCK != 2; }
__global__ void __launch_bounds__(CP_THREADS) k_mx4_dequantize_flat(long long R, int K, uint32_t magic,
                                                                    const uint32_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales,
                                                                    float* __restrict__ x) {
    const int nb = mx_blocks(K), nw = mx_words(K);
    const long long e0 = (long long)blockIdx.x * MXD_SPAN, row0 = e0 / K;  // the same for the block
    uint32_t k = (uint32_t)(e0 - row0 * K) + 4 * threadIdx.x;
    // (the magic number is exact: k < 2 MXD_SPAN here)
    const uint32_t r = K <= MXD_SPAN ? __umulhi(k, magic) : k >= (uint32_t)K;
    const long long row = row0 + r;
    if (row >= R) return;
    k -= r * K;
    const int over = (int)k + 4 - K;            // values of the next row, if any
    const bool more = over > 0 && row + 1 < R;  // there is one
    const uint32_t* w = codes + row * nw + (k >> 3);
    const uint8_t* sp = scales + row * nb + (k >> 5);
    const int first = over > 0 ? 4 - over : GSR_MX_BLOCK - (int)(k & 31u);  // values under the first scale (4 or more: all)
    const uint32_t w0 = w[0], w1 = (k & 7u) > 4u && (int)(k >> 3) + 1 < nw ? w[1] : 0u;
    const uint32_t next = more ? codes[(row + 1) * nw] : 0u;
    const float s0 = mx_scale(sp[0]), s1 = first < 4 && (over <= 0 || more) ? mx_scale(sp[1]) : 1.0f;
    uint32_t v = __funnelshift_r(w0, w1, 4 * (k & 7u));
    if (over > 0) v = (v & ((1u << 4 * (4 - over)) - 1u)) | next << 4 * (4 - over);
    const f2v a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v, s0, 0), b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v, s0, 1);
    const f2v a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v, s1, 0), b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v, s1, 1);
    const v4a o = {a0.x, first < 2 ? a1.y : a0.y, first < 3 ? b1.x : b0.x, first < 4 ? b1.y : b0.y};
    float* p = x + e0 + 4 * threadIdx.x;
    if (over <= 0 || more) {
        __builtin_nontemporal_store(o, reinterpret_cast<v4a*>(p));
    } else {  // the end of the tensor
        p[0] = o.x;
        if (over < 3) p[1] = o.y;
        if (over < 2) p[2] = o.z;
    }
}

// --------------------------------------------------------------------- colours --
// No contraction by the compiler from here on: the products that are to be fused say so, and so
// every kernel that evaluates an expression gets the same bits.
#pragma clang fp contract(off)
__device__ __forceinline__ float mad(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double mad(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Real spherical harmonics up to degree 3 in the reference's order and signs
// (utils/sh_utils.py:26-48): Y_k = SH_C[k] p_k(x, y, z), p_k the polynomials of sh_values.  The
// constants go into a Gaussian's coefficients once, not into every view's basis (8 views of 300k
// Gaussians at degree 3: 11.6 -> 10.7 us).
__device__ constexpr double SH_C[16] = {
    0.28209479177387814,
    -0.4886025119029199, 0.4886025119029199, -0.4886025119029199,
    1.0925484305920792, -1.0925484305920792, 0.31539156525252005, -1.0925484305920792, 0.5462742152960396,
    -0.5900435899266435, 2.890611442640554, -0.4570457994644658, 0.3731763325901154, -0.4570457994644658,
    1.445305721320277, -0.5900435899266435};

// p_k, k >= 1 (p_0 = 1); F = float, or double where a sign needs it.
template <int DEG, typename F>
__device__ __forceinline__ void sh_values(F x, F y, F z, F* b) {
    b[0] = (F)1;
    if constexpr (DEG > 0) {
        b[1] = y; b[2] = z; b[3] = x;
    }
    if constexpr (DEG > 1) {
        const F xx = x * x, yy = y * y, zz2 = (F)2 * (z * z), t = xx + yy, d = xx - yy;
        b[4] = x * y; b[5] = y * z; b[6] = zz2 - t; b[7] = x * z;
        b[8] = d;
        if constexpr (DEG > 2) {
            const F o = mad((F)2, zz2, -t);
            b[9] = y * mad((F)3, xx, -yy);
            b[10] = b[4] * z;
            b[11] = o * y;
            b[12] = z * mad((F)-3, t, zz2);
            b[13] = o * x;
            b[14] = z * d;
            b[15] = x * mad((F)-3, yy, xx);
        }
    }
}

// sum_k w[k] grad p_k at (x, y, z) (what they have along (x, y, z) itself drops out in the
// projection that follows).
template <int DEG>
__device__ __forceinline__ void sh_grad(float x, float y, float z, const float* w, float& gx, float& gy, float& gz) {
    gx = gy = gz = 0.0f;
    if constexpr (DEG > 0) {
        gx = w[3]; gy = w[1]; gz = w[2];
    }
    if constexpr (DEG > 1) {
        const float w6 = 2.0f * w[6], w8 = 2.0f * w[8];
        gx = mad(y, w[4], mad(z, w[7], mad(x, w8 - w6, gx)));
        gy = mad(x, w[4], mad(z, w[5], mad(-y, w8 + w6, gy)));
        gz = mad(y, w[5], mad(x, w[7], mad(2.0f * z, w6, gz)));
    }
    if constexpr (DEG > 2) {
        const float xx = x * x, yy = y * y, zz = z * z, xy = x * y, yz = y * z, xz = x * z, t = xx + yy, d = xx - yy;
        const float w9 = 3.0f * w[9], w12 = 3.0f * w[12], w15 = 3.0f * w[15], z4 = 4.0f * zz;
        gx = mad(2.0f * xy, w9 - w[11], gx);
        gx = mad(yz, w[10], gx);
        gx = mad(2.0f * xz, w[14] - w12, gx);
        gx = mad(z4 - mad(2.0f, xx, t), w[13], gx);
        gx = mad(d, w15, gx);
        gy = mad(d, w9, gy);
        gy = mad(xz, w[10], gy);
        gy = mad(z4 - mad(2.0f, yy, t), w[11], gy);
        gy = mad(-2.0f * yz, w12 + w[14], gy);
        gy = mad(-2.0f * xy, w[13] + w15, gy);
        gz = mad(xy, w[10], gz);
        gz = mad(8.0f * z, mad(y, w[11], x * w[13]), gz);
        gz = mad(mad(2.0f, zz, -t), w12, gz);
        gz = mad(d, w[14], gz);
    }
}

struct ShArgs {
    int P, V, pitch, nb, M;
    const float* xyz;
    const float* dc;
    long long dc_stride;
    const uint32_t* codes;
    const uint8_t* scales;
    const float* campos;
};

struct v3a {  // (a struct: a vector of three would be stored as four)
    float x, y, z;
};
__device__ __forceinline__ v3a load3(const float* p) { return {p[0], p[1], p[2]}; }
__device__ __forceinline__ void store3(float* p, float x, float y, float z) {
    p[0] = x; p[1] = y; p[2] = z;
}
__device__ __forceinline__ void store3_past(float* p, float x, float y, float z) {  // past the caches
    __builtin_nontemporal_store(x, p);
    __builtin_nontemporal_store(y, p + 1);
    __builtin_nontemporal_store(z, p + 2);
}

// Coefficients of one Gaussian, 3 floats each, coefficient 0 the constant one: decoded, then times
// SH_C (fold).  The codes stay for the sign in 64 bits.
template <int DEG>
struct Coef {
    static constexpr int N = (DEG + 1) * (DEG + 1);
    static constexpr int WORDS = (3 * (N - 1) + 7) / 8;   // code words that the degree needs
    static constexpr int BLOCKS = (3 * (N - 1) + GSR_MX_BLOCK - 1) / GSR_MX_BLOCK;
    float q[8 * WORDS + 3];   // q[0..2] as they are
    float base[3];            // 1/2 + Y_0 dc
    uint32_t w[WORDS + 1];
    uint32_t bytes;           // scales
    __device__ __forceinline__ float scale(int block) const { return mx_scale(bytes >> (8 * block) & 255u); }
    __device__ __forceinline__ void decode() {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) mx_decode8(w[j], scale(j / 4), q + 3 + 8 * j);
    }
    __device__ __forceinline__ void fold() {
#pragma unroll
        for (int j = 0; j < 3; ++j) base[j] = mad((float)SH_C[0], q[j], 0.5f);
#pragma unroll
        for (int k = 1; k < N; ++k)
#pragma unroll
            for (int j = 0; j < 3; ++j) q[3 * k + j] *= (float)SH_C[k];
    }
    __device__ __forceinline__ void load(int i, const ShArgs& a) {
        const v3a d = a.dc ? load3(a.dc + i * a.dc_stride) : v3a{0.0f, 0.0f, 0.0f};
        q[0] = d.x; q[1] = d.y; q[2] = d.z;
#pragma unroll
        for (int k = 0; k < WORDS; ++k) w[k] = a.codes[(long long)i * a.pitch + k];
        bytes = 0;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) bytes |= (uint32_t)a.scales[(long long)i * a.nb + k] << (8 * k);
        decode();
    }
    // The value before the clamp for basis polynomials b: smallest terms first.
    __device__ __forceinline__ void sum(const float* b, float* s) const {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            float t = 0.0f;
#pragma unroll
            for (int k = N - 1; k >= 1; --k) t = mad(b[k], q[3 * k + j], t);
            s[j] = t + base[j];
        }
    }
};

// u -> u / |u|; returns 1 / |u|, 0 (and d = 0) where u is 0.
__device__ __forceinline__ float normalize3(float& x, float& y, float& z) {
    float n = mad(x, x, mad(y, y, z * z)), back = 1.0f;
    if (__builtin_expect(!(n > 1e-30f && n < 1e30f), 0)) {  // the squares leave the range (or u is 0, or not finite)
        const float m = fmaxf(fabsf(x), fmaxf(fabsf(y), fabsf(z)));
        const bool some = m > 0.0f;
        const float by = some ? m : 1.0f;
        x /= by; y /= by; z /= by;
        n = some ? mad(x, x, mad(y, y, z * z)) : 1.0f;
        back = some ? 1.0f / m : 0.0f;
    }
    // the hardware's reciprocal root (good to 2 units of 2^-24) and a Newton step: a third of the
    // instructions of a rounded root and quotient
    float r = __builtin_amdgcn_rsqf(n);
    r *= mad(-0.5f * n * r, r, 1.5f);
    x *= r; y *= r; z *= r;
    return r * back;
}

// The value before the clamp in 64 bits, from the codes.
template <int DEG>
__device__ __forceinline__ void preclamp64(const Coef<DEG>& c, v3a p, float cx, float cy, float cz, double* s) {
    constexpr int N = Coef<DEG>::N;
    const double x = (double)p.x - cx, y = (double)p.y - cy, z = (double)p.z - cz;
    const double n = x * x + y * y + z * z;
    const double r = n > 0.0 ? 1.0 / sqrt(n) : 0.0;
    double b[N];
    sh_values<DEG, double>(x * r, y * r, z * r, b);
#pragma unroll
    for (int j = 0; j < 3; ++j) s[j] = mad(SH_C[0], (double)c.q[j], 0.5);
#pragma unroll
    for (int m = 0; m < Coef<DEG>::WORDS; ++m) {
        float v[8];
        uint32_t w = c.w[m];
        asm volatile("" : "+v"(w));  // decoded here, not kept in registers through the views
        mx_decode8(w, c.scale(m / 4), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int f = 8 * m + e + 3, k = f / 3;
            if (k < N) s[f % 3] = mad(SH_C[k] * b[k], (double)v[e], s[f % 3]);
        }
    }
}

// Colours of one Gaussian in every view; with MASK, which channels the clamp lets through (a
// byte a view).  Rounding of the value before the clamp, in units of 2^-24: a direction is good to
// 6, a basis value (slope at most 4.9) to 37, the sum of 16 products to 53 of the coefficients'
// sum; nearer to zero than 64 the sign is taken from 64 bits, so that no gradient hangs on a
// rounding.
template <int DEG, bool MASK, bool NT>
__device__ __forceinline__ void write_colors(const ShArgs& a, int i, v3a p, Coef<DEG>& c,
                                             float* __restrict__ colors, uint8_t* __restrict__ mask) {
    float near[3] = {0.5f, 0.5f, 0.5f};
    if constexpr (MASK) {
#pragma unroll
        for (int k = 0; k < Coef<DEG>::N; ++k)
#pragma unroll
            for (int j = 0; j < 3; ++j) near[j] += fabsf(c.q[3 * k + j]);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) near[j] *= 0x1p-18f;
    c.fold();
    float cx = a.campos[0], cy = a.campos[1], cz = a.campos[2];
    for (int v = 0; v < a.V; ++v) {
        const float* ahead = a.campos + (v + 1 < a.V ? 3 * v + 3 : 0);  // the next camera, while this one's colours are made
        const float nx = ahead[0], ny = ahead[1], nz = ahead[2];
        float x = p.x - cx, y = p.y - cy, z = p.z - cz;
        normalize3(x, y, z);
        float b[Coef<DEG>::N], s[3];
        sh_values<DEG, float>(x, y, z, b);
        c.sum(b, s);
        if constexpr (MASK) {
            bool on[3], close = false;
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                on[j] = s[j] >= 0.0f;
                close |= fabsf(s[j]) < near[j];
            }
            if (close) {
                double t[3];
                preclamp64<DEG>(c, p, cx, cy, cz, t);
#pragma unroll
                for (int j = 0; j < 3; ++j) on[j] = t[j] >= 0.0;
            }
            mask[(long long)v * a.P + i] = (uint8_t)(on[0] | on[1] << 1 | on[2] << 2);
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] = s[j] < 0.0f ? 0.0f : s[j];  // keeps a NaN
        float* o = colors + ((long long)v * a.P + i) * 3;
        if constexpr (NT) store3_past(o, s[0], s[1], s[2]);
        else store3(o, s[0], s[1], s[2]);
        cx = nx; cy = ny; cz = nz;
    }
}

// Colours from 16 MB on, a sixteenth of the 256 MB cache, pass by the caches: write-back of their lines stands in the way of
// reads.  Both sides, through and past, with inputs that change from pass to pass and with the same ones again: 8 views of 300k
// Gaussians (28.8 MB) 13.4 and 10.3, 12.0 and 9.2 us; of 175k (16.8 MB) 8.3 and 7.2, 8.3 and 7.0; of 130k (12.5 MB) 7.1 and 6.1,
// 6.5 and 5.9; one view of 4M (48 MB) 44.0 and 41.4, 34.4 and 34.5; of 1M (12 MB) 13.3 and 12.5, 10.9 and 11.4.  From 16 MB on
// the kernel is as fast or faster past them, while the next reader of the colours pays 5 to 25 % for it (a pass right behind 8
// views of 250k: both together 20.2 and 21.1, 22.0 and 20.8; behind 1M 19.7 and 19.5, 16.2 and 17.0).  Their gradients are read
// through the caches at any size (past them, backward of 1M with 4 views 48 -> 62 us).
constexpr long long NT_COLOR_BYTES = 16LL << 20;

// One thread per Gaussian, its coefficients in registers for all views.  Bound by memory with
// one view (62 bytes a Gaussian at degree 3), by the vector units with many.
template <int DEG, bool MASK, bool NT>
__global__ void __launch_bounds__(CP_THREADS) k_sh_colors(ShArgs a, float* __restrict__ colors,
                                                          uint8_t* __restrict__ mask) {
    const int i = blockIdx.x * CP_THREADS + threadIdx.x;
    if (i >= a.P) return;
    const v3a p = load3(a.xyz + 3LL * i);
    Coef<DEG> c;
    c.load(i, a);
    write_colors<DEG, MASK, NT>(a, i, p, c, colors, mask);
}

// ---- rows of features through LDS ------------------------------------------------
// A wave's 64 rows of 3 M floats lie in one piece of memory, a lane works on one row: the piece
// moves as float4s of consecutive lanes and turns in the wave's own part of LDS (no block
// barrier: a wave's LDS operations are in order, a wait for them is enough).  M = 16: rows 13
// float4s apart, which spreads a lane-per-row access over all banks; other M: rows as they lie.
constexpr int ROW16 = 13;                  // float4s
constexpr int ROWS_LDS = 64 * 4 * ROW16;   // floats a wave (also 64 rows of 45)
__device__ __forceinline__ void wave_lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// With NT rows of 48 floats pass by the caches (the others, F != 48, go through them whatever NT says).  Both sides,
// through and past, one view.  Loads (forward), inputs that change: 58 MB of features (300k Gaussians) 18.8 and 15.3 us, 115 MB 32.5 and
// 28.6, 192 MB 62.0 and 45.6; the same inputs again: 58 MB 13.3 and 14.6, 96 MB 19.5 and 21.7, 154 MB 43.9 and 32.6, as the
// pass no longer fits the 256 MB cache.  In training every step goes through parameters, gradients and two moments, five
// times the features: from 52 MB of features on that is more than the cache holds, and the first case is the nearer one.
// Stores (the gradient): 29 MB 8.2 and 7.7, 8.5 and 7.7 with the same inputs; 58 MB 15.8 and 14.0, 13.5 and 12.9; 192 MB 45.1
// and 42.7, 45.3 and 40.9.  No crossing here either; a reader right behind pays 17 % at 58 MB, forward,
// backward and reader together 53.0 and 54.6, at 19 MB 23.5 and 23.6.  32 MB: an eighth of the cache.
constexpr long long NT_LOAD_BYTES = 64LL << 20, NT_STORE_BYTES = 32LL << 20;
template <bool NT>
__device__ __forceinline__ void rows_in(const float* __restrict__ src, int rows, int F, float* lds, int lane) {
    if (F == 48) {
        v4a v[12];
#pragma unroll
        for (int r = 0; r < 12; ++r) {
            const int f = lane + 64 * r;
            const v4a* q = reinterpret_cast<const v4a*>(src + 4 * f);
            v[r] = v4a{0.0f, 0.0f, 0.0f, 0.0f};
            if (f / 12 < rows) {
                if constexpr (NT) v[r] = __builtin_nontemporal_load(q);
                else v[r] = *q;
            }
        }
        float4* d = reinterpret_cast<float4*>(lds);
#pragma unroll
        for (int r = 0; r < 12; ++r) {
            const int f = lane + 64 * r;
            d[f / 12 * ROW16 + f % 12] = make_float4(v[r].x, v[r].y, v[r].z, v[r].w);
        }
    } else {
        const int n = (rows < 64 ? rows : 64) * F;
        for (int f = 4 * lane; f < n; f += 256) {
            const v4a v = load4(src + f, f, n);
            *reinterpret_cast<float4*>(lds + f) = make_float4(v.x, v.y, v.z, v.w);
        }
    }
    wave_lds_wait();
}

template <bool NT>
__device__ __forceinline__ void rows_out(float* __restrict__ dst, int rows, int F, const float* lds, int lane) {
    wave_lds_wait();
    if (F == 48) {
        const float4* d = reinterpret_cast<const float4*>(lds);
#pragma unroll
        for (int r = 0; r < 12; ++r) {
            const int f = lane + 64 * r;
            const float4 v = d[f / 12 * ROW16 + f % 12];
            v4a* q = reinterpret_cast<v4a*>(dst + 4 * f);
            const v4a o = {v.x, v.y, v.z, v.w};
            if (f / 12 < rows) {
                if constexpr (NT) __builtin_nontemporal_store(o, q);
                else *q = o;
            }
        }
    } else {
        const int n = (rows < 64 ? rows : 64) * F;
        for (int f = 4 * lane; f < n; f += 256) {
            const float4 v = *reinterpret_cast<const float4*>(lds + f);
            if (f + 4 <= n) {
                *reinterpret_cast<v4a*>(dst + f) = v4a{v.x, v.y, v.z, v.w};
            } else {
                dst[f] = v.x;
                if (f + 1 < n) dst[f + 1] = v.y;
                if (f + 2 < n) dst[f + 2] = v.z;
            }
        }
    }
}

// Training forward: a Gaussian's fp32 coefficients are read once, rounded to codes (kept for the
// backward), read back and evaluated.  Bound by memory: 1M Gaussians at degree 3 with 4 views (282 MB) 52 us,
// 5.4 TB/s.  The blocks that the degree touches are rounded whole, so a
// code does not depend on the degree.
template <int DEG, bool NT, bool NT_COLOR>
__global__ void __launch_bounds__(CP_THREADS) k_sh_colors_quantize(ShArgs a, const float* __restrict__ features,
                                                                   uint32_t* __restrict__ codes,
                                                                   uint8_t* __restrict__ scales,
                                                                   uint8_t* __restrict__ mask,
                                                                   float* __restrict__ colors) {
    using C = Coef<DEG>;
    __shared__ float4 s_rows[CP_THREADS / 64][ROWS_LDS / 4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = blockIdx.x * CP_THREADS + wave * 64, i = first + lane, F = 3 * a.M;
    if (first >= a.P) return;  // the whole wave
    float* lds = reinterpret_cast<float*>(s_rows[wave]);
    rows_in<NT>(features + (long long)first * F, a.P - first, F, lds, lane);
    if (i >= a.P) return;
    constexpr int VALUES = C::BLOCKS * GSR_MX_BLOCK;  // of the row behind its constant coefficient
    float v[VALUES + 3];
    if (F == 48) {
        const float4* d = reinterpret_cast<const float4*>(lds) + lane * ROW16;
#pragma unroll
        for (int k = 0; k < 12; ++k) {
            const float4 t = d[k];
            const float e[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * k + j < VALUES + 3) v[4 * k + j] = e[j];
        }
#pragma unroll
        for (int k = 48; k < VALUES + 3; ++k) v[k] = 0.0f;
    } else {
#pragma unroll
        for (int k = 0; k < VALUES + 3; ++k) v[k] = k < F ? lds[lane * F + k] : 0.0f;
    }
    const v3a p = load3(a.xyz + 3LL * i);
    C c;
    c.q[0] = v[0]; c.q[1] = v[1]; c.q[2] = v[2];
    c.bytes = 0;
#pragma unroll
    for (int b = 0; b < C::BLOCKS; ++b) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < GSR_MX_BLOCK; ++k) {
            const uint32_t x = __float_as_uint(v[3 + b * GSR_MX_BLOCK + k]) & 0x7FFFFFFFu;
            m = m > x ? m : x;
        }
        const uint32_t sb = mx_scale_byte(m);
        c.bytes |= sb << (8 * b);
#pragma unroll
        for (int j = 4 * b; j < 4 * b + 4; ++j)
            if (j < C::WORDS) {
                const float* x = v + 3 + 8 * j;
                c.w[j] = sb == 255u ? 0u : mx_encode8(v4a{x[0], x[1], x[2], x[3]}, v4a{x[4], x[5], x[6], x[7]},
                                                      mx_scale(sb));
            }
    }
    c.decode();
#pragma unroll
    for (int j = 0; j < C::WORDS; ++j) codes[(long long)i * a.pitch + j] = c.w[j];
#pragma unroll
    for (int b = 0; b < C::BLOCKS; ++b) scales[(long long)i * a.nb + b] = (uint8_t)(c.bytes >> (8 * b));
    write_colors<DEG, true, NT_COLOR>(a, i, p, c, colors, mask);
}

// One thread per Gaussian, all views; the features' gradient rows leave through LDS.  Which
// channels take part comes from the forward's mask, so the constant coefficients (whose basis value
// has no slope) are not read.
// WANT_F: dfeatures is wanted (else at most its first coefficient, ddc).  Bound by memory: 1M Gaussians at
// degree 3 with 4 views (294 MB) 49 us, 6.0 TB/s.
template <int DEG, bool WANT_F, bool NT>
__global__ void __launch_bounds__(CP_THREADS) k_sh_colors_backward(ShArgs a, const uint8_t* __restrict__ mask,
                                                                   const float* __restrict__ dcolors,
                                                                   float* __restrict__ dxyz, float* __restrict__ ddc,
                                                                   float* __restrict__ dfeatures) {
    constexpr int N = Coef<DEG>::N, NF = WANT_F ? N : 1;
    __shared__ float4 s_rows[WANT_F ? CP_THREADS / 64 : 1][WANT_F ? ROWS_LDS / 4 : 1];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = blockIdx.x * CP_THREADS + wave * 64;
    if (first >= a.P) return;                                 // the whole wave
    const int i = first + lane < a.P ? first + lane : a.P - 1;  // lanes behind the end repeat the last row
    const v3a p = load3(a.xyz + 3LL * i);
    Coef<DEG> c;
    c.load(i, a);
    c.fold();
    float acc[3 * NF];
#pragma unroll
    for (int k = 0; k < 3 * NF; ++k) acc[k] = 0.0f;
    float ax = 0.0f, ay = 0.0f, az = 0.0f;
    for (int v = 0; v < a.V; ++v) {
        const float* cam = a.campos + 3 * v;
        const v3a gp = load3(dcolors + ((long long)v * a.P + i) * 3);
        const uint32_t on = mask[(long long)v * a.P + i];
        float x = p.x - cam[0], y = p.y - cam[1], z = p.z - cam[2];
        const float r = normalize3(x, y, z);
        float b[N];
        sh_values<DEG, float>(x, y, z, b);
        const float g[3] = {on & 1u ? gp.x : 0.0f, on & 2u ? gp.y : 0.0f, on & 4u ? gp.z : 0.0f};
#pragma unroll
        for (int k = 0; k < NF; ++k)
#pragma unroll
            for (int j = 0; j < 3; ++j) acc[3 * k + j] = mad(b[k], g[j], acc[3 * k + j]);
        if (DEG > 0 && dxyz) {
            float w[N], gx, gy, gz;
#pragma unroll
            for (int k = 1; k < N; ++k)
                w[k] = mad(c.q[3 * k], g[0], mad(c.q[3 * k + 1], g[1], c.q[3 * k + 2] * g[2]));
            sh_grad<DEG>(x, y, z, w, gx, gy, gz);
            const float along = mad(gx, x, mad(gy, y, gz * z));
            ax = mad(r, mad(-along, x, gx), ax);
            ay = mad(r, mad(-along, y, gy), ay);
            az = mad(r, mad(-along, z, gz), az);
        }
    }
#pragma unroll
    for (int k = 0; k < 3 * NF; ++k) acc[k] *= (float)SH_C[k / 3];
    if (first + lane < a.P) {
        if (dxyz) store3(dxyz + 3LL * i, ax, ay, az);
        if (ddc) store3(ddc + 3LL * i, acc[0], acc[1], acc[2]);
    }
    if constexpr (WANT_F) {
        const int F = 3 * a.M;
        float* lds = reinterpret_cast<float*>(s_rows[wave]);
        if (F == 48) {
            float4* d = reinterpret_cast<float4*>(lds) + lane * ROW16;
            auto at = [&](int k) { return k < 3 * N ? acc[k] : 0.0f; };
#pragma unroll
            for (int k = 0; k < 12; ++k) d[k] = make_float4(at(4 * k), at(4 * k + 1), at(4 * k + 2), at(4 * k + 3));
        } else {
#pragma unroll
            for (int k = 0; k < 3 * N; ++k) lds[lane * F + k] = acc[k];
            for (int k = 3 * N; k < F; ++k) lds[lane * F + k] = 0.0f;
        }
        rows_out<NT>(dfeatures + (long long)first * F, a.P - first, F, lds, lane);
    }
}

// Bound by memory: 12 bytes a row, or the 20 that a column of a [P, 3] gradient fetches (what its caller has); one thread
// each (a column has nothing wide to load).  1M rows 3.8 us, of a column 4.7.
__global__ void __launch_bounds__(CP_THREADS) k_accumulate_weights(int P, const float* __restrict__ w,
                                                                   long long stride, float decay,
                                                                   float* __restrict__ acc) {
    const int i = blockIdx.x * CP_THREADS + threadIdx.x;
    if (i < P) acc[i] = mad(decay, acc[i], w[i * stride]);
}

// -------------------------------------------------------------------- eviction --
// The rows to keep of a group are its last `recent` ones and the heaviest `pick` of those
// before them.  Radix selection: three histogram passes (11, 11, 10 bits from the top) find the
// key T of the pick-th heaviest row and how many of the rows equal to it are kept (`ties`, the
// lowest first); then the ids are written in order.  Every count is an integer, so the result
// does not depend on the order of the atomics.
//   One block per group does it all for groups of up to KEEP_SMALL rows, the keys in registers;
// larger groups take a launch per pass, the last of which also counts for each tile what the kernel
// that writes the ids needs: what is read, 4 bytes a row and pass from the caches, is less than what
// the launches and their dependences cost (five launches; 1M rows 26 us, with a sixth for the counts 29).
constexpr int KEEP_TILE = CP_THREADS * 16;  // rows a block holds at once
constexpr int KEEP_BINS = 2048;
constexpr int KEEP_SMALL_THREADS = 1024, KEEP_SMALL = KEEP_SMALL_THREADS * 16;

struct KeepGroup {
    int begin, end, old_end;  // rows [begin, old_end) compete, [old_end, end) are kept
    int pick;
    int out;    // first output slot
    int tile0;  // first tile
};
struct KeepArgs {
    int n, tiles, rounds;
    KeepGroup g[GSR_KEEP_MAX_GROUPS];
};
struct KeepSel {
    uint32_t prefix, need;  // digits found so far; the rank looked for among the keys that share them
    uint32_t count;         // how many those are
};
struct KeepWs {
    uint32_t* hist;  // [groups][3][KEEP_BINS]
    KeepSel* sel;    // [groups][3]
    uint32_t* above; // [tiles] rows above the first 22 bits of T (with those that share them, if all of them stay)
    uint16_t* from;  // [tiles][KEEP_LOW] rows that share them with low bits of at least the index
};
constexpr int KEEP_LOW = 1024;  // the last pass's bins
// A block takes so many times KEEP_TILE rows of a group (a tile) that there are about 1024 tiles: fewer
// histograms to add up, and what the last kernel reads of the tiles before its own grows with their
// square (10M rows, one piece a tile and three: 130 -> 80 us; 45M, one and eleven: 702 -> 183; 3M, one and
// two: 47 -> 41 with the weights in the caches, but an eviction with its rows 181 -> 184, so one).
// At most 15: a tile's counts are kept in 16 bits.
inline int keep_rounds(size_t P) {
    const size_t r = (P / KEEP_TILE + 1023) / 1024;
    return (int)(r < 1 ? 1 : r > 15 ? 15 : r);
}
inline size_t keep_tiles(size_t P) { return P / ((size_t)KEEP_TILE * keep_rounds(P)) + GSR_KEEP_MAX_GROUPS + 1; }
inline size_t keep_hist_bytes() { return (size_t)GSR_KEEP_MAX_GROUPS * 3 * KEEP_BINS * 4; }
inline KeepWs keep_ws(void* p, size_t tiles) {
    char* c = static_cast<char*>(p);
    KeepWs w;
    w.hist = reinterpret_cast<uint32_t*>(c);
    w.sel = reinterpret_cast<KeepSel*>(c + keep_hist_bytes());
    c += keep_hist_bytes() + align_up(GSR_KEEP_MAX_GROUPS * 3 * sizeof(KeepSel));
    w.above = reinterpret_cast<uint32_t*>(c);
    w.from = reinterpret_cast<uint16_t*>(c + align_up(tiles * sizeof(uint32_t)));
    return w;
}

// Weights in the order of unsigned integers: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t keep_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = w == 0.0f ? 0u : __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int keep_group_of(const KeepArgs& a, int tile) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (a.g[m].tile0 <= tile) lo = m;
        else hi = m - 1;
    }
    return lo;
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {  // inclusive, DPP row shifts and broadcasts
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
    return x;
}

// Exclusive scan over the block's threads; every thread calls it, each time with an s_wave that no
// thread still reads.
template <int THREADS>
__device__ __forceinline__ uint32_t block_scan_excl(uint32_t x, uint32_t* s_wave) {
    const uint32_t inc = wave_scan(x);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) s_wave[wave] = inc;
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) base += w < wave ? s_wave[w] : 0u;
    return base + inc - x;
}

// The bin, counted from the top, that holds the need-th largest key, and the rank inside it
// (need >= 1 and at most the sum of the bins).
template <int THREADS>
__device__ __forceinline__ KeepSel find_bin(const uint32_t* hist, uint32_t need, uint32_t* s_wave, KeepSel* s_out) {
    constexpr int PER = KEEP_BINS / THREADS;
    const int top = KEEP_BINS - 1 - (int)threadIdx.x * PER;
    uint32_t h[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += h[k] = hist[top - k];
    uint32_t above = block_scan_excl<THREADS>(sum, s_wave);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        if (above < need && need <= above + h[k]) *s_out = {(uint32_t)(top - k), need - above, h[k]};
        above += h[k];
    }
    __syncthreads();
    return *s_out;
}

// A thread's N keys are all the same: they are added as one (adds to one counter queue, and equal
// weights are common: 10k rows of zeros 34 -> 10 us, 1M 33 -> 27, 45M 577 -> 179; different ones cost 0.2 more).
template <int N>
__device__ __forceinline__ bool keep_flat(const uint32_t (&key)[N], bool all_in) {
    uint32_t x = 0;
#pragma unroll
    for (int k = 1; k < N; ++k) x |= key[k] ^ key[0];
    return x == 0 && all_in;
}

// Keys [i, i + N) of rows below `end` (behind it that of 0.0: every reader goes by the row).
template <int N>
__device__ __forceinline__ void keep_load(const float* __restrict__ w, long long i, long long end, uint32_t (&key)[N]) {
    v4a v[N / 4];
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        v[q] = v4a{0.0f, 0.0f, 0.0f, 0.0f};
        if (i + 4 * q + 4 <= end) {
            v[q] = *reinterpret_cast<const v4a*>(w + i + 4 * q);
        } else {
            if (i + 4 * q < end) v[q].x = w[i + 4 * q];
            if (i + 4 * q + 1 < end) v[q].y = w[i + 4 * q + 1];
            if (i + 4 * q + 2 < end) v[q].z = w[i + 4 * q + 2];
        }
    }
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        key[4 * q] = keep_key(v[q].x); key[4 * q + 1] = keep_key(v[q].y);
        key[4 * q + 2] = keep_key(v[q].z); key[4 * q + 3] = keep_key(v[q].w);
    }
}

template <int PASS>
__device__ __forceinline__ bool keep_digit(uint32_t key, uint32_t prefix, uint32_t& d) {
    d = PASS == 0 ? key >> 21 : PASS == 1 ? (key >> 10) & 2047u : key & 1023u;
    return PASS == 0 || (PASS == 1 ? key >> 21 : key >> 10) == prefix;
}

// All rows that share the 22 bits found in two passes stay: T is just below them, without ties.
__device__ __forceinline__ bool keep_early(KeepSel st) { return st.count == st.need && st.prefix > 0; }

// One pass over the keys of a small group: the digits found before it -> one more.
template <int PASS, int N>
__device__ __forceinline__ KeepSel keep_small_pass(const uint32_t (&key)[N], bool flat, int n, KeepSel st, uint32_t* h,
                                                   uint32_t* s_wave, KeepSel* s_out) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        uint32_t d;
        const bool in = keep_digit<PASS>(key[k], st.prefix, d) && (int)threadIdx.x * N + k < n;
        if (in && (k == 0 || !flat)) atomicAdd(&h[d], flat ? (uint32_t)N : 1u);
    }
    __syncthreads();
    const KeepSel b = find_bin<KEEP_SMALL_THREADS>(h, st.need, s_wave, s_out);
    return {(st.prefix << (PASS == 2 ? 10 : 11)) | b.prefix, b.need, b.count};
}

// Bound by latency: one load of the keys, two or three rounds of LDS counters and scans behind it.  N keys a
// thread, as few as the largest group allows, so that all 16 waves share the work: 1000 rows 4.0 us (with 16 a
// thread 8.0), 4000 4.5 (7.0), 10k 7.5 (8.5).  More than 16 are no gain over the launches of the large way (32k
// rows 25 us, 17 there).
template <int N>
__global__ void __launch_bounds__(KEEP_SMALL_THREADS) k_keep_small(KeepArgs a, const float* __restrict__ w,
                                                                   int* __restrict__ ids) {
    // a part for each pass: no barrier between one pass's last reads and the next one's first writes
    __shared__ uint32_t h[3][KEEP_BINS];
    __shared__ uint32_t s_wave[4][KEEP_SMALL_THREADS / 64];
    __shared__ KeepSel s_out[3];
    const KeepGroup G = a.g[blockIdx.x];
    const int n = G.old_end - G.begin, first = threadIdx.x * N;
    if (G.pick > 0) {  // the whole block
        uint32_t key[N];
        keep_load(w, (long long)G.begin + first, G.old_end, key);
        for (int k = threadIdx.x; k < 3 * KEEP_BINS; k += KEEP_SMALL_THREADS) h[0][k] = 0u;
        __syncthreads();
        const bool flat = keep_flat(key, first + N <= n);
        KeepSel st = {0u, (uint32_t)G.pick, 0u};
        st = keep_small_pass<0>(key, flat, n, st, h[0], s_wave[0], &s_out[0]);
        st = keep_small_pass<1>(key, flat, n, st, h[1], s_wave[1], &s_out[1]);
        if (keep_early(st)) {
            st.prefix = (st.prefix << 10) - 1;
            st.need = 0;
        } else {
            st = keep_small_pass<2>(key, flat, n, st, h[2], s_wave[2], &s_out[2]);
        }
        uint32_t gt = 0, eq = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            gt += first + k < n && key[k] > st.prefix;
            eq += first + k < n && key[k] == st.prefix;
        }
        const uint32_t before = block_scan_excl<KEEP_SMALL_THREADS>(gt | eq << 16, s_wave[3]);  // at most KEEP_SMALL < 65536 each
        gt = before & 0xFFFFu;
        eq = before >> 16;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (first + k < n) {
                const bool up = key[k] > st.prefix, tie = key[k] == st.prefix;
                if (up || (tie && eq < st.need)) ids[G.out + gt + (eq < st.need ? eq : st.need)] = G.begin + first + k;
                gt += up;
                eq += tie;
            }
        }
    }
    for (int k = threadIdx.x; k < G.end - G.old_end; k += KEEP_SMALL_THREADS) ids[G.out + G.pick + k] = G.old_end + k;
}

__global__ void __launch_bounds__(CP_THREADS) k_keep_clear(uint32_t* __restrict__ p, int n) {
    for (int i = blockIdx.x * CP_THREADS + threadIdx.x; i < n; i += gridDim.x * CP_THREADS) p[i] = 0u;
}

// Digits found before pass PASS of group g: the first tile's block leaves them for the later
// kernels, every block works them out for itself.
template <int PASS>
__device__ __forceinline__ KeepSel keep_state(const KeepArgs& a, const KeepWs& ws, int g, int tile, uint32_t* s_wave,
                                              KeepSel* s_out) {
    KeepSel prev = {0u, (uint32_t)a.g[g].pick, 0u};
    if constexpr (PASS == 0) return prev;
    if (PASS > 1) prev = ws.sel[g * 3 + PASS - 2];
    const KeepSel b = find_bin<CP_THREADS>(ws.hist + ((size_t)g * 3 + PASS - 1) * KEEP_BINS, prev.need, s_wave, s_out);
    const KeepSel now = {(prev.prefix << (PASS == 3 ? 10 : 11)) | b.prefix, b.need, b.count};
    if (PASS < 3 && tile == a.g[g].tile0 && threadIdx.x == 0) ws.sel[g * 3 + PASS - 1] = now;
    return now;
}

// LAST: the rows above the 22 bits are counted for each tile, and those that share them by their low bits
// (running sums from the top, so that the next kernel reads two numbers a tile whatever T is) -- or
// with the others, if all of them stay.
// MANY: more than one piece a tile (the loop costs 1M rows, which are one each, 27.7 us instead of 26.1).
template <int PASS, bool MANY>
__global__ void __launch_bounds__(CP_THREADS) k_keep_hist(KeepArgs a, KeepWs ws, const float* __restrict__ w) {
    constexpr bool LAST = PASS == 2;
    constexpr int BINS = LAST ? KEEP_LOW : KEEP_BINS;
    __shared__ uint32_t h[BINS];
    __shared__ uint32_t s_wave[3][CP_THREADS / 64];
    __shared__ KeepSel s_out;
    const int tile = blockIdx.x, g = keep_group_of(a, tile);
    const KeepGroup G = a.g[g];
    if (G.pick == 0) return;  // nothing to look for (the whole block)
    uint32_t key[16];
    const int rounds = MANY ? a.rounds : 1;
    long long base = G.begin + (long long)(tile - G.tile0) * rounds * KEEP_TILE + threadIdx.x * 16;
    keep_load(w, base, G.old_end, key);
    for (int k = threadIdx.x; k < BINS; k += CP_THREADS) h[k] = 0u;
    const KeepSel st = keep_state<PASS>(a, ws, g, tile, s_wave[0], &s_out);
    __syncthreads();
    const bool early = LAST && keep_early(st);
    uint32_t above = 0;
    for (int round = 1;; ++round) {
        const bool flat = keep_flat(key, base + 16 <= G.old_end);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            uint32_t d;
            const bool in = base + k < G.old_end, same = keep_digit<PASS>(key[k], st.prefix, d);
            if constexpr (LAST) above += in && (key[k] >> 10 > st.prefix || (same && early));
            if (in && same && !early && (k == 0 || !flat)) atomicAdd(&h[d], flat ? 16u : 1u);
        }
        base += KEEP_TILE;
        if (!MANY || round == rounds || base - threadIdx.x * 16 >= G.old_end) break;  // the whole block
        keep_load(w, base, G.old_end, key);
    }
    if constexpr (LAST) {
        const uint32_t before = block_scan_excl<CP_THREADS>(above, s_wave[1]);
        if (threadIdx.x == CP_THREADS - 1) ws.above[tile] = before + above;
        if (early) return;  // the whole block
    }
    __syncthreads();
    uint32_t* out = ws.hist + ((size_t)g * 3 + PASS) * KEEP_BINS;
    for (int k = threadIdx.x; k < BINS; k += CP_THREADS)
        if (h[k]) atomicAdd(&out[k], h[k]);
    if constexpr (LAST) {
        const int first = KEEP_LOW - 4 - 4 * (int)threadIdx.x;  // four bins a thread, from the top
        const uint32_t h3 = h[first + 3], h2 = h3 + h[first + 2], h1 = h2 + h[first + 1], h0 = h1 + h[first];
        const uint32_t b = block_scan_excl<CP_THREADS>(h0, s_wave[2]);
        const uint32_t lo = (b + h0) | (b + h1) << 16, hi = (b + h2) | (b + h3) << 16;
        *reinterpret_cast<uint2*>(ws.from + (size_t)tile * KEEP_LOW + first) = make_uint2(lo, hi);
    }
}

// A tile's kept rows: ranked by a scan over the threads (16 rows each, in order), gathered in LDS
// and written in one piece behind those of the tiles before.
template <bool MANY>
__global__ void __launch_bounds__(CP_THREADS) k_keep_write(KeepArgs a, KeepWs ws, const float* __restrict__ w,
                                                           int* __restrict__ ids) {
    __shared__ uint32_t s_wave[2][CP_THREADS / 64];
    __shared__ uint32_t s_gt, s_eq;
    __shared__ int s_ids[KEEP_TILE];
    __shared__ uint32_t s_n;
    __shared__ KeepSel s_out;
    const int tile = blockIdx.x, g = keep_group_of(a, tile);
    const KeepGroup G = a.g[g];
    const int rounds = MANY ? a.rounds : 1;
    const long long span = (long long)rounds * KEEP_TILE, base = G.begin + (tile - G.tile0) * span;
    if (G.pick > 0 && base < G.old_end) {  // the whole block
        long long first = base + threadIdx.x * 16;
        uint32_t key[16];
        keep_load(w, first, G.old_end, key);
        KeepSel st = ws.sel[g * 3 + 1];
        if (threadIdx.x == 0) s_gt = s_eq = 0;
        uint2 sum = {0u, 0u};
        for (int t = G.tile0 + threadIdx.x; t < tile; t += CP_THREADS) sum.x += ws.above[t];
        if (keep_early(st)) {
            st = {(st.prefix << 10) - 1, 0u, 0u};
            __syncthreads();
        } else {
            st = keep_state<3>(a, ws, g, tile, s_wave[0], &s_out);  // (its barriers order s_gt and s_eq too)
            const uint32_t low = st.prefix & (KEEP_LOW - 1);
            for (int t = G.tile0 + threadIdx.x; t < tile; t += CP_THREADS) {
                const uint16_t* f = ws.from + (size_t)t * KEEP_LOW + low;
                const uint32_t up = low + 1 < KEEP_LOW ? f[1] : 0u;
                sum.x += up;
                sum.y += f[0] - up;
            }
        }
        sum.x = wave_scan(sum.x);
        sum.y = wave_scan(sum.y);
        if ((threadIdx.x & 63) == 63) {
            atomicAdd(&s_gt, sum.x);
            atomicAdd(&s_eq, sum.y);
        }
        uint32_t gt0 = 0, eq0 = 0;  // rows above / equal to T before this piece
        for (int round = 1;; ++round) {
            uint32_t both = 0;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (first + k < G.old_end) both += key[k] > st.prefix ? 1u : key[k] == st.prefix ? 1u << 16 : 0u;
            const uint32_t before = block_scan_excl<CP_THREADS>(both, s_wave[1]);
            if (round == 1) {  // (the scan's barrier also ends the sum)
                gt0 = s_gt;
                eq0 = s_eq;
            }
            const uint32_t ties = eq0 < st.need ? st.need - eq0 : 0u;  // left for this piece
            uint32_t gt = before & 0xFFFFu, eq = before >> 16;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (first + k < G.old_end) {
                    const bool up = key[k] > st.prefix, tie = key[k] == st.prefix;
                    if (up || (tie && eq < ties)) s_ids[gt + (eq < ties ? eq : ties)] = (int)(first + k);
                    gt += up;
                    eq += tie;
                }
            }
            if (threadIdx.x == CP_THREADS - 1) s_n = gt | eq << 16;  // at most KEEP_TILE = 4096 of each
            first += KEEP_TILE;
            const bool more = MANY && round < rounds && first - threadIdx.x * 16 < G.old_end;  // the whole block
            if (more) keep_load(w, first, G.old_end, key);
            __syncthreads();
            gt = s_n & 0xFFFFu;
            eq = s_n >> 16;
            int* out = ids + G.out + gt0 + (eq0 < st.need ? eq0 : st.need);
            for (uint32_t k = threadIdx.x; k < gt + (eq < ties ? eq : ties); k += CP_THREADS) out[k] = s_ids[k];
            if (!more) break;
            gt0 += gt;  // (the next scan's barrier is behind all reads of s_ids and s_n)
            eq0 += eq;
        }
    }
    const long long lo = base > G.old_end ? base : G.old_end, hi = base + span < G.end ? base + span : G.end;
    for (long long i = lo + threadIdx.x; i < hi; i += CP_THREADS) ids[G.out + G.pick + (i - G.old_end)] = (int)i;
}

// ------------------------------------------------------------------------ rows --
// A copy: K rows of each tensor read and written once, bound by memory.  A block moves
// TAKE_SPAN units of one tensor's output, a unit being 16 bytes where the rows are whole and aligned
// float4s (the features, 48 of a Gaussian's 61 floats, and the rotations), else the largest of 12, 8 and
// 4 that a row is made of (with 4 for all of those, their blocks were 40 % of the launch for 15 % of the
// bytes).  All loads, and the stores of 16 and 12 bytes, pass by the caches: a line is wanted by
// one instruction.  1M rows of 732 bytes kept at 70 %: 181 us, 5.7 TB/s of what has to move; with units of 16
// and 4 bytes only 196, with temporal accesses 215.  Narrow rows cost the lines of their dropped neighbours too.
constexpr int TAKE_MAX = 32;    // tensors a launch
// Units a thread: their ids, then their values, are in flight together.  3: a block is 64 rows of 192 bytes,
// whole cache lines (2: 184 us, 4: 182, 8: 197).
constexpr int TAKE_PER = 3;
constexpr int TAKE_SPAN = CP_THREADS * TAKE_PER;
struct TakeTensor {
    const void* src;
    void* dst;
    Tiling t;
    int K;  // rows to write (0 where they are 0 wide)
    int rows, vec, pad;
    uint32_t block0, blocks;  // first block, how many
};
struct TakeArgs {
    int n;
    TakeTensor t[TAKE_MAX];
};

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
template <int U>
struct TakeUnit {
    uint32_t w[U];
};
template <int U>
__device__ __forceinline__ TakeUnit<U> take_load(const uint32_t* p) {
    TakeUnit<U> v;
    if constexpr (U == 4) {
        const u4v q = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(p));
        v.w[0] = q.x; v.w[1] = q.y; v.w[2] = q.z; v.w[3] = q.w;
    } else {
#pragma unroll
        for (int k = 0; k < U; ++k) v.w[k] = __builtin_nontemporal_load(p + k);
    }
    return v;
}
template <int U>
__device__ __forceinline__ void take_store(uint32_t* p, const TakeUnit<U>& v) {
    if constexpr (U == 4) {
        __builtin_nontemporal_store(u4v{v.w[0], v.w[1], v.w[2], v.w[3]}, reinterpret_cast<u4v*>(p));
    } else {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if constexpr (U == 3) __builtin_nontemporal_store(v.w[k], p + k);
            else p[k] = v.w[k];
        }
    }
}
template <int U>
__device__ __forceinline__ void take_block(const TakeTensor& t, uint32_t block, const int* __restrict__ ids) {
    const uint32_t* src = static_cast<const uint32_t*>(t.src);
    uint32_t* dst = static_cast<uint32_t*>(t.dst);
    long long to[TAKE_PER], from[TAKE_PER];
#pragma unroll
    for (int k = 0; k < TAKE_PER; ++k) {
        long long row;
        int unit;
        to[k] = from[k] = -1;
        if (tiling_place<TAKE_SPAN>(t.t, block, k * CP_THREADS + threadIdx.x, t.K, row, unit)) {
            to[k] = (row * t.t.units + unit) * U;
            const int id = ids[row];
            if ((unsigned)id < (unsigned)t.rows) from[k] = ((long long)id * t.t.units + unit) * U;
        }
    }
    TakeUnit<U> v[TAKE_PER] = {};
#pragma unroll
    for (int k = 0; k < TAKE_PER; ++k)
        if (from[k] >= 0) v[k] = take_load<U>(src + from[k]);
#pragma unroll
    for (int k = 0; k < TAKE_PER; ++k)
        if (to[k] >= 0) take_store<U>(dst + to[k], v[k]);
    if (t.pad > 0 && block == t.blocks - 1) {  // the words behind the last row
        uint32_t* tail = dst + (long long)t.K * t.t.units * U;
        for (int k = threadIdx.x; k < t.pad; k += CP_THREADS) tail[k] = 0u;
    }
}

__global__ void __launch_bounds__(CP_THREADS) k_take_rows(TakeArgs a, const int* __restrict__ ids) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (a.t[m].block0 <= blockIdx.x) lo = m;
        else hi = m - 1;
    }
    const TakeTensor t = a.t[lo];
    const uint32_t block = blockIdx.x - t.block0;
    if (t.vec == 4) take_block<4>(t, block, ids);
    else if (t.vec == 3) take_block<3>(t, block, ids);
    else if (t.vec == 2) take_block<2>(t, block, ids);
    else take_block<1>(t, block, ids);
}

unsigned grid_for(long long items, long long cap) {
    const long long g = (items + CP_THREADS - 1) / CP_THREADS;
    return (unsigned)(g < 1 ? 1 : g > cap ? cap : g);
}

// A launch has fewer than 2^32 threads.
constexpr long long MAX_BLOCKS = ((1LL << 32) - 1) / CP_THREADS;

// One thread per Gaussian, its index an int: the last block's must not pass 2^31.
constexpr int MAX_P = 0x7FFFFFFF - CP_THREADS;

// Does a weight lie in the memory of a sum that is not its own?  (That sum is written before it is read, or after.)
bool shared_apart(int P, const float* weights, long long stride, const float* acc) {
    if (weights == acc && (stride == 1 || P == 1)) return false;
    typedef __int128 wide;  // addresses in bytes: no product leaves it
    wide step = 4 * (wide)stride, w = (wide)(uintptr_t)weights;
    const wide a = (wide)(uintptr_t)acc, end = a + 4 * (wide)P;
    const bool back = step < 0;
    if (back) {  // from the other end
        w += step * (P - 1);
        step = -step;
    }
    const wide i = w + 4 > a ? 0 : step > 0 ? (a - w - 4) / step + 1 : P;  // the first weight that ends behind acc
    if (i >= P || w + i * step >= end) return false;
    const bool only = i + 1 == P || w + (i + 1) * step >= end;
    return !only || w + i * step != a + 4 * (back ? P - 1 - i : i);
}

int check_rows(long long R, int K) {
    if (R < 0 || K < 0 || K > GSR_MAX_WIDTH || (K > 0 && R > (1LL << 42) / K))  // (products of the two stay far from 2^63)
        return set_error("[gsr] mx4: invalid number or width of rows");
    return 0;
}

int check_colors(int P, int V, int degree, int M, const float* xyz, const float* dc, const uint32_t* codes,
                 const uint8_t* scales, const float* campos) {
    if (P < 0 || P > MAX_P || V < 1 || V > GSR_MAX_VIEWS)
        return set_error("[gsr] sh_colors: invalid P or number of views");
    if (degree < 0 || degree > 3 || M < (degree + 1) * (degree + 1) || M > 16)
        return set_error("[gsr] sh_colors: degree must be 0..3 with (degree + 1)^2 <= M <= 16");
    if (P > 0 && (!xyz || !dc || !campos || (M > 1 && (!codes || !scales))))
        return set_error("[gsr] sh_colors: null buffer");
    return 0;
}

ShArgs sh_args(int P, int V, int M, const float* xyz, const float* dc, long long dc_stride, const uint32_t* codes,
               const uint8_t* scales, const float* campos) {
    return {P, V, mx_words(3 * (M - 1)), mx_blocks(3 * (M - 1)), M, xyz, dc, dc_stride, codes, scales, campos};
}

}  // namespace
}  // namespace gsr

using namespace gsr;

extern "C" {

GSR_API int gsr_mx4_quantize(long long R, int K, const float* x, long long row_stride, uint32_t* codes,
                             uint8_t* scales, void* stream) {
    if (int rc = check_rows(R, K)) return rc;
    if (R == 0 || K == 0) return 0;
    if (!x || !codes || !scales) return set_error("[gsr] gsr_mx4_quantize: null buffer");
    if (row_stride < K && R > 1) return set_error("[gsr] gsr_mx4_quantize: rows overlap");
    const Tiling t = tiling(mx_blocks(K), MXQ_SPAN);
    const long long blocks = tiling_blocks(t, R, MXQ_SPAN);
    if (blocks > MAX_BLOCKS) return set_error("[gsr] gsr_mx4_quantize: too many rows in one call");
    k_mx4_quantize<<<(unsigned)blocks, CP_THREADS, 0, (hipStream_t)stream>>>(R, K, t, x, row_stride, codes, scales);
    return launched("mx4_quantize");
}

GSR_API int gsr_mx4_dequantize(long long R, int K, const uint32_t* codes, const uint8_t* scales, float* x,
                               void* stream) {
    if (int rc = check_rows(R, K)) return rc;
    if (R == 0 || K == 0) return 0;
    if (!x || !codes || !scales) return set_error("[gsr] gsr_mx4_dequantize: null buffer");
    if (mxd_flat(K)) {
        const long long blocks = (R * K + MXD_SPAN - 1) / MXD_SPAN;
        if (blocks > MAX_BLOCKS) return set_error("[gsr] gsr_mx4_dequantize: too many rows in one call");
        k_mx4_dequantize_flat<<<(unsigned)blocks, CP_THREADS, 0, (hipStream_t)stream>>>(
            R, K, (uint32_t)((1ULL << 32) / K + 1), codes, scales, x);
        return launched("mx4_dequantize");
    }
    const Tiling t = tiling((K + 3) / 4, CP_THREADS);
    const long long blocks = tiling_blocks(t, R, CP_THREADS);
    if (blocks > MAX_BLOCKS) return set_error("[gsr] gsr_mx4_dequantize: too many rows in one call");
    k_mx4_dequantize<<<(unsigned)blocks, CP_THREADS, 0, (hipStream_t)stream>>>(
        R, K, t, reinterpret_cast<const uint16_t*>(codes), scales, x);
    return launched("mx4_dequantize");
}

GSR_API int gsr_sh_colors(int P, int V, int degree, int M, const float* xyz, const float* dc, long long dc_stride,
                          const uint32_t* codes, const uint8_t* scales, const float* campos, float* colors,
                          uint8_t* mask, void* stream) {
    if (int rc = check_colors(P, V, degree, M, xyz, dc, codes, scales, campos)) return rc;
    if (P == 0) return 0;
    if (!colors) return set_error("[gsr] gsr_sh_colors: null buffer");
    const ShArgs a = sh_args(P, V, M, xyz, dc, dc_stride, codes, scales, campos);
    const unsigned grid = grid_for(P, 1LL << 31);
    hipStream_t st = (hipStream_t)stream;
    const bool past = 12LL * P * V > NT_COLOR_BYTES;
#define GSR_SH_COLORS(D)                                                                       \
    if (mask && past) k_sh_colors<D, true, true><<<grid, CP_THREADS, 0, st>>>(a, colors, mask); \
    else if (mask) k_sh_colors<D, true, false><<<grid, CP_THREADS, 0, st>>>(a, colors, mask);   \
    else if (past) k_sh_colors<D, false, true><<<grid, CP_THREADS, 0, st>>>(a, colors, nullptr); \
    else k_sh_colors<D, false, false><<<grid, CP_THREADS, 0, st>>>(a, colors, nullptr)
    if (degree == 0) { GSR_SH_COLORS(0); }
    else if (degree == 1) { GSR_SH_COLORS(1); }
    else if (degree == 2) { GSR_SH_COLORS(2); }
    else { GSR_SH_COLORS(3); }
#undef GSR_SH_COLORS
    return launched("sh_colors");
}

GSR_API int gsr_sh_colors_quantize(int P, int V, int degree, int M, const float* xyz, const float* features,
                                   const float* campos, uint32_t* codes, uint8_t* scales, uint8_t* mask,
                                   float* colors, void* stream) {
    if (int rc = check_colors(P, V, degree, M, xyz, features, codes, scales, campos)) return rc;
    if (P == 0) return 0;
    if (!mask || !colors) return set_error("[gsr] gsr_sh_colors_quantize: null buffer");
    const ShArgs a = sh_args(P, V, M, xyz, nullptr, 0, nullptr, nullptr, campos);
    const unsigned grid = grid_for(P, 1LL << 31);
    hipStream_t st = (hipStream_t)stream;
    const bool nt = 12LL * M * P > NT_LOAD_BYTES;
    const bool past = 12LL * P * V > NT_COLOR_BYTES;
#define GSR_SH_QUANTIZE_AS(...) \
    k_sh_colors_quantize<__VA_ARGS__><<<grid, CP_THREADS, 0, st>>>(a, features, codes, scales, mask, colors)
#define GSR_SH_QUANTIZE(D)                            \
    if (nt && past) GSR_SH_QUANTIZE_AS(D, true, true); \
    else if (nt) GSR_SH_QUANTIZE_AS(D, true, false);   \
    else if (past) GSR_SH_QUANTIZE_AS(D, false, true); \
    else GSR_SH_QUANTIZE_AS(D, false, false)
    if (degree == 0) { GSR_SH_QUANTIZE(0); }
    else if (degree == 1) { GSR_SH_QUANTIZE(1); }
    else if (degree == 2) { GSR_SH_QUANTIZE(2); }
    else { GSR_SH_QUANTIZE(3); }
#undef GSR_SH_QUANTIZE
#undef GSR_SH_QUANTIZE_AS
    return launched("sh_colors_quantize");
}

GSR_API int gsr_sh_colors_backward(int P, int V, int degree, int M, const float* xyz, const uint32_t* codes,
                                   const uint8_t* scales, const float* campos, const uint8_t* mask,
                                   const float* dcolors, float* dxyz, float* ddc, float* dfeatures, void* stream) {
    if (int rc = check_colors(P, V, degree, M, xyz, xyz, codes, scales, campos)) return rc;
    if (P == 0 || (!dxyz && !ddc && !dfeatures)) return 0;
    if (!mask || !dcolors) return set_error("[gsr] gsr_sh_colors_backward: null buffer");
    const ShArgs a = sh_args(P, V, M, xyz, nullptr, 0, codes, scales, campos);
    const unsigned grid = grid_for(P, 1LL << 31);
    hipStream_t st = (hipStream_t)stream;
    const bool nt = 12LL * M * P > NT_STORE_BYTES;
#define GSR_SH_BACKWARD_AS(...) \
    k_sh_colors_backward<__VA_ARGS__><<<grid, CP_THREADS, 0, st>>>(a, mask, dcolors, dxyz, ddc, dfeatures)
#define GSR_SH_BACKWARD(D)                              \
    if (!dfeatures) GSR_SH_BACKWARD_AS(D, false, false); \
    else if (nt) GSR_SH_BACKWARD_AS(D, true, true);      \
    else GSR_SH_BACKWARD_AS(D, true, false)
    if (degree == 0) { GSR_SH_BACKWARD(0); }
    else if (degree == 1) { GSR_SH_BACKWARD(1); }
    else if (degree == 2) { GSR_SH_BACKWARD(2); }
    else { GSR_SH_BACKWARD(3); }
#undef GSR_SH_BACKWARD
#undef GSR_SH_BACKWARD_AS
    return launched("sh_colors_backward");
}

GSR_API int gsr_accumulate_weights(int P, const float* weights, long long stride, float decay, float* acc,
                                   void* stream) {
    if (P < 0 || P > MAX_P) return set_error("[gsr] gsr_accumulate_weights: invalid P");
    if (P == 0) return 0;
    if (!weights || !acc) return set_error("[gsr] gsr_accumulate_weights: null buffer");
    if (shared_apart(P, weights, stride, acc))
        return set_error("[gsr] gsr_accumulate_weights: the weights overlap the sums, element on another element");
    k_accumulate_weights<<<grid_for(P, 1LL << 31), CP_THREADS, 0, (hipStream_t)stream>>>(P, weights, stride, decay, acc);
    return launched("accumulate_weights");
}

GSR_API size_t gsr_keep_ws_bytes(int P) {
    if (P <= KEEP_SMALL) return 0;  // no group is larger
    return keep_hist_bytes() + align_up(GSR_KEEP_MAX_GROUPS * 3 * sizeof(KeepSel)) +
           align_up(keep_tiles((size_t)P) * sizeof(uint32_t)) + keep_tiles((size_t)P) * KEEP_LOW * sizeof(uint16_t);
}

GSR_API int gsr_keep_heaviest(int P, const float* weights, int n_groups, const gsr_keep_group* groups, int* ids,
                              void* ws, void* stream) {
    if (P < 0 || n_groups < 0 || n_groups > GSR_KEEP_MAX_GROUPS)
        return set_error("[gsr] gsr_keep_heaviest: at most " + std::to_string(GSR_KEEP_MAX_GROUPS) + " groups a call");
    if (n_groups > 0 && !groups) return set_error("[gsr] gsr_keep_heaviest: null groups");
    KeepArgs a{};
    a.rounds = keep_rounds((size_t)P);
    const long long span = (long long)KEEP_TILE * a.rounds;
    int last = 0, most = 0;
    long long out = 0;
    for (int g = 0; g < n_groups; ++g) {
        const gsr_keep_group& q = groups[g];
        if (q.begin < last || q.end < q.begin || q.end > P)
            return set_error("[gsr] gsr_keep_heaviest: groups must be ascending ranges of rows that do not overlap");
        if (q.keep < 0 || q.keep > q.end - q.begin || q.recent < 0 || q.recent > q.keep)
            return set_error("[gsr] gsr_keep_heaviest: 0 <= recent <= keep <= rows of the group");
        last = q.end;
        if (q.keep == 0) continue;  // nothing to write
        a.g[a.n++] = {q.begin, q.end, q.end - q.recent, q.keep - q.recent, (int)out, a.tiles};
        a.tiles += (int)((q.end - q.begin + span - 1) / span);
        out += q.keep;
        most = std::max(most, q.end - q.begin);
    }
    if (a.n == 0) return 0;
    if (!weights || !ids || (!ws && P > KEEP_SMALL)) return set_error("[gsr] gsr_keep_heaviest: null buffer");
    hipStream_t st = (hipStream_t)stream;
    if (most <= KEEP_SMALL) {
        const int each = (most + KEEP_SMALL_THREADS - 1) / KEEP_SMALL_THREADS;  // keys a thread
        if (each <= 4) k_keep_small<4><<<a.n, KEEP_SMALL_THREADS, 0, st>>>(a, weights, ids);
        else if (each <= 8) k_keep_small<8><<<a.n, KEEP_SMALL_THREADS, 0, st>>>(a, weights, ids);
        else if (each <= 12) k_keep_small<12><<<a.n, KEEP_SMALL_THREADS, 0, st>>>(a, weights, ids);
        else k_keep_small<16><<<a.n, KEEP_SMALL_THREADS, 0, st>>>(a, weights, ids);
        return launched("keep_heaviest");
    }
    const KeepWs w = keep_ws(ws, keep_tiles((size_t)P));
    const int words = a.n * 3 * KEEP_BINS;
    k_keep_clear<<<grid_for(words, 1024), CP_THREADS, 0, st>>>(w.hist, words);
#define GSR_KEEP(MANY)                                                       \
    k_keep_hist<0, MANY><<<a.tiles, CP_THREADS, 0, st>>>(a, w, weights);      \
    k_keep_hist<1, MANY><<<a.tiles, CP_THREADS, 0, st>>>(a, w, weights);      \
    k_keep_hist<2, MANY><<<a.tiles, CP_THREADS, 0, st>>>(a, w, weights);      \
    k_keep_write<MANY><<<a.tiles, CP_THREADS, 0, st>>>(a, w, weights, ids)
    if (a.rounds > 1) { GSR_KEEP(true); }
    else { GSR_KEEP(false); }
#undef GSR_KEEP
    return launched("keep_heaviest");
}

GSR_API int gsr_take_rows(int K, const int* ids, int n, const gsr_rows* tensors, void* stream) {
    if (K < 0 || n < 0 || (n > 0 && !tensors) || (K > 0 && n > 0 && !ids))
        return set_error("[gsr] gsr_take_rows: invalid arguments");
    for (int k = 0; k < n; ++k) {
        const gsr_rows& t = tensors[k];
        if (t.width < 0 || t.width > GSR_MAX_WIDTH || t.rows < 0 || t.pad < 0)
            return set_error("[gsr] gsr_take_rows: invalid width or rows");
        const long long words = (long long)K * t.width;
        if ((words > 0 && t.rows > 0 && !t.src) || (words + t.pad > 0 && !t.dst))
            return set_error("[gsr] gsr_take_rows: null buffer");
    }
    // what is written is neither read nor written by another tensor of the call
    struct Range {
        uintptr_t lo, hi;
        bool meets(const Range& o) const { return lo < hi && o.lo < o.hi && lo < o.hi && o.lo < hi; }
    };
    auto written = [&](const gsr_rows& t) -> Range {
        return {(uintptr_t)t.dst, (uintptr_t)t.dst + 4 * ((uintptr_t)K * t.width + t.pad)};
    };
    for (int k = 0; k < n; ++k) {
        const Range w = written(tensors[k]);
        bool clash = w.meets({(uintptr_t)ids, (uintptr_t)ids + 4 * (uintptr_t)K});
        for (int j = 0; j < n; ++j) {
            const gsr_rows& t = tensors[j];
            clash |= w.meets({(uintptr_t)t.src, (uintptr_t)t.src + 4 * (uintptr_t)t.rows * t.width});
            clash |= j != k && w.meets(written(t));
        }
        if (clash) return set_error("[gsr] gsr_take_rows: a destination overlaps the ids or another tensor of the call");
    }
    // the tensors of a launch: their blocks, or -1 where a launch does not hold them
    auto launch_of = [&](int k0, TakeArgs& a) -> long long {
        long long blocks = 0;
        for (int k = k0; k < n && k < k0 + TAKE_MAX; ++k) {
            const gsr_rows& q = tensors[k];
            const bool wide = q.width % 4 == 0 && ((uintptr_t)q.src | (uintptr_t)q.dst) % 16 == 0;
            const int unit = wide ? 4 : q.width % 3 == 0 ? 3 : q.width % 2 == 0 ? 2 : 1;  // words
            if ((long long)K * q.width + q.pad == 0) continue;
            const Tiling t = tiling(std::max(1, q.width / unit), TAKE_SPAN);
            const int rows = q.width > 0 ? K : 0;
            const long long nb = std::max(1LL, tiling_blocks(t, rows, TAKE_SPAN));
            a.t[a.n++] = {q.src, q.dst, t, rows, q.rows, unit, q.pad, (uint32_t)blocks, (uint32_t)nb};
            blocks += nb;
            if (blocks > MAX_BLOCKS) return -1;
        }
        return blocks;
    };
    hipStream_t st = (hipStream_t)stream;
    TakeArgs a{};
    long long blocks = launch_of(0, a);
    bool fits = blocks >= 0;
    for (int k0 = TAKE_MAX; k0 < n && fits; k0 += TAKE_MAX) {  // (before the first launch)
        TakeArgs later{};
        fits = launch_of(k0, later) >= 0;
    }
    if (!fits) return set_error("[gsr] gsr_take_rows: too many rows in one call");
    bool any = false;
    for (int k0 = 0; k0 < n; k0 += TAKE_MAX) {
        if (k0 > 0) {
            a = TakeArgs{};
            blocks = launch_of(k0, a);
        }
        if (a.n == 0) continue;
        any = true;
        k_take_rows<<<(unsigned)blocks, CP_THREADS, 0, st>>>(a, ids);
    }
    return any ? launched("take_rows") : 0;
}

}  // extern "C"
