// Rows in 8 bits (definition: lowbit.h): a cache of rows that are quantised as they are written, and a linear layer that keeps
// its input in 8 bits for its backward.
#include "lowbit.h"

namespace {

// the two halves of a word as numbers of a 16-bit type
template <typename T> __device__ __forceinline__ float low16(unsigned w)
{
    if constexpr (__is_same(T, LbF16)) return (float)__builtin_bit_cast(_Float16, (unsigned short)w);
    else return __uint_as_float(w << 16);
}
template <typename T> __device__ __forceinline__ float high16(unsigned w)
{
    if constexpr (__is_same(T, LbF16)) return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
    else return __uint_as_float(w & 0xffff0000u);
}

// ------------------------------------------------------------------ row cache
// Both directions move 16 bytes of the caller's rows per lane and step (COLS = 4 float32 or 8 16-bit numbers, neighbouring lanes
// neighbouring addresses, at any alignment: gfx950 loads and stores 16 bytes from any address) and their codes as one word or two.
// FULL: width is a multiple of COLS, so that no lane has a shorter share (1 M x 256 float32 read back: 217 us, without 327).
// Bound by memory: 1 M x 256 float32 is written in 273 to 279 us (4.7 TB/s of rows and codes, a copy's rate) and read in 214 to 217; 333 k
// scattered rows of 64 are read in 25 us (4.5 TB/s).  Odd widths (5, 17, 257) are written at 2.5 to 4.4 TB/s and read at 2.9 to 3.3.
// A workgroup owns rpb rows, i.e. about ROWS8_ITEMS (row, columns) items; item e of it is row e / cpr by a multiply-high (exact:
// e * cpr < 2^32).
#define ROWS8_ITEMS 2048
#define ROWS8_ROWS 256

// the maximum over the 2^shift neighbouring lanes of a group (uniform): four steps within 16 lanes, then across
__device__ __forceinline__ unsigned group_max(unsigned m, int shift)
{
    if (shift > 0) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));    // lane ^ 1
    if (shift > 1) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));    // lane ^ 2
    if (shift > 2) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));   // mirrored in 8
    if (shift > 3) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, true));   // mirrored in 16
    if (shift > 4) m = max(m, (unsigned)__shfl_xor((int)m, 16, 64));
    return m;
}

// where lanes read that must not read past the end of a caller's array
__device__ const uint4 kZeroPage[2] = {};

template <typename T> __device__ __forceinline__ uint4 load16(const T* p)
{
    uint4 w;
    __builtin_memcpy(&w, p, 16);
    return w;
}

template <int FMT, typename T, typename S, bool FULL>
__global__ __launch_bounds__(256) void rows8_write_kernel(gs4d_rows8 c, const T* __restrict__ rows, long long ld, long long n,
                                                          const S* __restrict__ slots, long long start, int cpr, int rpb, unsigned rcp, int lshift, int dup)
{
    constexpr int COLS = 16 / (int)sizeof(T);
    __shared__ long long s_slot[ROWS8_ROWS];
    const long long i0 = (long long)blockIdx.x * rpb;
    const int nrow = (int)min((long long)rpb, n - i0);
    // few rows at given slots are one per workgroup, whose lanes look whether a later row has the same slot
    bool later = false;
    if (dup == 1) later = __syncthreads_or((int)threadIdx.x < n && (int)threadIdx.x > i0 && slots[min((int)threadIdx.x, (int)n - 1)] == slots[i0]);
    // where each row of this workgroup goes (-1: nowhere): one lane per row
    if ((int)threadIdx.x < nrow) {
        const long long i = i0 + threadIdx.x;
        long long slot = slots ? (long long)slots[i] : start + i;
        if (slot < 0 || slot >= c.capacity || later) slot = -1;
        if (dup == 2 && slot >= 0) {
            // rows8_owner_kernel left the last row's number.  It leaves the word zero again: a row that reads it later is not
            // the last one either way
            if (c.owner[slot] == (int)(i + 1)) c.owner[slot] = 0;
            else slot = -1;
        }
        s_slot[threadIdx.x] = slot;
    }
    __syncthreads();
    const int items = nrow * cpr, ng = (c.width + c.group - 1) / c.group;
    constexpr int U = 4;
    const T* end = rows + (n - 1) * ld + c.width;
    for (int e0 = threadIdx.x; e0 < items; e0 += 256 * U) {
        uint4 w[U];
        int ch[U];
        long long slot[U];
        const T* x[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int e = min(e0 + 256 * u, items - 1);
            const int r = cpr == 1 ? e : (int)__umulhi((unsigned)e, rcp);
            ch[u] = e - r * cpr;
            slot[u] = e0 + 256 * u < items ? s_slot[r] : -1;
            // the last columns of a row are read with what follows them, those of the array's last row one by one (below)
            x[u] = rows + (i0 + r) * ld + ch[u] * COLS;
            // (FULL: a group's columns past the width are read from the row's last ones instead)
            if (FULL) w[u] = load16(x[u] - max(ch[u] * COLS - (c.width - COLS), 0));
            else w[u] = load16(x[u] + COLS <= end ? x[u] : reinterpret_cast<const T*>(kZeroPage));
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float v[COLS];
            if (!FULL && x[u] + COLS > end) {
#pragma unroll
                for (int q = 0; q < COLS; q++) v[q] = x[u] + q < end ? lb_load(x[u][q]) : 0.f;
            } else {
                const unsigned e[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
                for (int q = 0; q < COLS; q++) {
                    if constexpr (sizeof(T) == 4) v[q] = __uint_as_float(e[q]);
                    else v[q] = (q & 1) ? high16<T>(e[q >> 1]) : low16<T>(e[q >> 1]);
                }
            }
#pragma unroll
            for (int q = 0; q < COLS; q++) v[q] = ch[u] * COLS + (FULL ? 0 : q) < c.width ? v[q] : 0.f;
            unsigned m = 0;
#pragma unroll
            for (int q = 0; q < COLS; q++) m = max(m, lb_abs_bits(v[q]));
            const LbScale sc = lb_scale<FMT>(group_max(m, lshift));
            const int col = ch[u] * COLS;
            if (slot[u] < 0 || col >= c.width) continue;
            unsigned* out = reinterpret_cast<unsigned*>(c.codes + (size_t)slot[u] * c.pitch + col);
            const unsigned w0 = lb_encode4<FMT>(v[0] * sc.inv, v[1] * sc.inv, v[2] * sc.inv, v[3] * sc.inv);
            if constexpr (COLS == 8)
                *reinterpret_cast<uint2*>(out) = make_uint2(w0, lb_encode4<FMT>(v[4] * sc.inv, v[5] * sc.inv, v[6] * sc.inv, v[7] * sc.inv));
            else
                *out = w0;
            if ((ch[u] & ((1 << lshift) - 1)) == 0) c.scales[(size_t)slot[u] * ng + (ch[u] >> lshift)] = sc.s;
        }
    }
}

// Many scattered rows: the last row of a slot is found by a maximum over row numbers (order of arrival does not matter)
template <typename S>
__global__ __launch_bounds__(256) void rows8_owner_kernel(gs4d_rows8 c, const S* __restrict__ slots, long long n)
{
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long slot = slots[i];
    if (slot >= 0 && slot < c.capacity) atomicMax(c.owner + slot, (int)(i + 1));
}

template <int FMT, typename T, typename S, bool FULL>
__global__ __launch_bounds__(256) void rows8_read_kernel(gs4d_rows8 c, T* __restrict__ out, long long ld, long long n,
                                                         const S* __restrict__ slots, long long start, int cpr, int rpb, unsigned rcp, int gshift)
{
    constexpr int COLS = 16 / (int)sizeof(T);
    __shared__ long long s_slot[ROWS8_ROWS];
    const long long i0 = (long long)blockIdx.x * rpb;
    const int nrow = (int)min((long long)rpb, n - i0);
    if ((int)threadIdx.x < nrow) {
        const long long slot = slots ? (long long)slots[i0 + threadIdx.x] : start + i0 + threadIdx.x;
        s_slot[threadIdx.x] = slot >= 0 && slot < c.capacity ? slot : -1;
    }
    __syncthreads();
    const int items = nrow * cpr, ng = (c.width + c.group - 1) / c.group;
    constexpr int U = 4;
    for (int e0 = threadIdx.x; e0 < items; e0 += 256 * U) {
        unsigned w[U][2];
        float s[U];
        int row[U], col[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int e = min(e0 + 256 * u, items - 1);
            row[u] = cpr == 1 ? e : (int)__umulhi((unsigned)e, rcp);
            col[u] = (e - row[u] * cpr) * COLS;
            const long long slot = s_slot[row[u]];
            const size_t at = slot < 0 ? 0 : (size_t)slot;
            const unsigned char* p = c.codes + at * c.pitch + col[u];
            if constexpr (COLS == 8) { const uint2 t = *reinterpret_cast<const uint2*>(p); w[u][0] = t.x; w[u][1] = t.y; }
            else w[u][0] = *reinterpret_cast<const unsigned*>(p);
            s[u] = c.scales[at * ng + (col[u] >> gshift)];
            if (slot < 0) { w[u][0] = 0; w[u][1] = 0; s[u] = 0.f; }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (e0 + 256 * u >= items) break;
            T* y = out + (i0 + row[u]) * ld + col[u];
            const float4 a = lb_decode4<FMT>(w[u][0]);
            T o[COLS] = {lb_store<T>(s[u] * a.x), lb_store<T>(s[u] * a.y), lb_store<T>(s[u] * a.z), lb_store<T>(s[u] * a.w)};
            if constexpr (COLS == 8) {
                const float4 b = lb_decode4<FMT>(w[u][1]);
                o[4] = lb_store<T>(s[u] * b.x); o[5] = lb_store<T>(s[u] * b.y); o[6] = lb_store<T>(s[u] * b.z); o[7] = lb_store<T>(s[u] * b.w);
            }
            if (FULL || col[u] + COLS <= c.width) {
                __builtin_memcpy(y, o, 16);
            } else {
#pragma unroll
                for (int q = 0; q < COLS - 1; q++)
                    if (col[u] + q < c.width) y[q] = o[q];
            }
        }
    }
}

// ------------------------------------------------------------------ several matrices of rows at once (Gs4dKeepJobs)
// blockIdx.y: a group of 64 columns of one of the matrices; 16 lanes of 4 columns each, 64 rows per workgroup.  Bound by memory: 5 M rows
// of 1000 columns are packed in 4.9 ms and unpacked in 5.1 (about 5 TB/s of both sides).
template <bool WRITE>
__global__ __launch_bounds__(256) void keep_jobs_kernel(Gs4dKeepJobs jobs, long long rows)
{
    int job_v = 0;
    while (job_v + 1 < jobs.n && (int)blockIdx.y >= jobs.group0[job_v + 1]) job_v++;
    const int job = __builtin_amdgcn_readfirstlane(job_v);
    const Gs4dKeepJob& J = jobs.j[job];
    const int g = blockIdx.y - jobs.group0[job], ng = jobs.group0[job + 1] - jobs.group0[job], sub = threadIdx.x & 15, col = g * 64 + 4 * sub;
    const bool inside = col < J.width;
    constexpr int U = 4;
    const long long r0 = (long long)blockIdx.x * (16 * U) + (threadIdx.x >> 4);
    if (WRITE) {
        float4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = min(r0 + 16 * u, rows - 1);
            v[u] = *reinterpret_cast<const float4*>(J.x + r * J.ld + (inside ? col : 0));
            if (!inside) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = r0 + 16 * u;
            float e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            unsigned bits = 0, m = 0;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (J.relu) {
                    bits |= (e[q] > 0.f ? 1u : 0u) << (4 * (sub & 7) + q);
                    e[q] = e[q] < 0.f ? 0.f : e[q];
                }
                m = max(m, lb_abs_bits(e[q]));
            }
            m = group_max(m, 4);
            unsigned w;
            float s;
            if (J.relu) {
                const LbScale sc = lb_scale<GS4D_FMT_UINT8>(m);
                w = lb_encode4<GS4D_FMT_UINT8>(e[0] * sc.inv, e[1] * sc.inv, e[2] * sc.inv, e[3] * sc.inv);
                s = sc.s;
#pragma unroll
                for (int k = 1; k < 8; k <<= 1) bits |= (unsigned)__shfl_xor((int)bits, k, 64);
            } else {
                const LbScale sc = lb_scale<GS4D_FMT_INT8>(m);
                w = lb_encode4<GS4D_FMT_INT8>(e[0] * sc.inv, e[1] * sc.inv, e[2] * sc.inv, e[3] * sc.inv);
                s = sc.s;
            }
            if (r >= rows) continue;
            *reinterpret_cast<unsigned*>(J.codes + (r * ng + g) * 64 + 4 * sub) = w;
            if (sub == 0) J.scales[r * ng + g] = s;
            if (J.relu && (sub & 7) == 0) J.bits[(r * ng + g) * 2 + (sub >> 3)] = bits;
        }
    } else {
        unsigned w[U], bits[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = min(r0 + 16 * u, rows - 1);
            w[u] = *reinterpret_cast<const unsigned*>(J.codes + (r * ng + g) * 64 + 4 * sub);
            s[u] = J.scales[r * ng + g];
            bits[u] = J.relu ? J.bits[(r * ng + g) * 2 + (sub >> 3)] : 0u;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = r0 + 16 * u;
            float4 v = J.relu ? lb_decode4<GS4D_FMT_UINT8>(w[u]) : lb_decode4<GS4D_FMT_INT8>(w[u]);
            v = make_float4(s[u] * v.x, s[u] * v.y, s[u] * v.z, s[u] * v.w);
            if (J.relu) {                                 // a positive number whose code is 0 stays positive: the sign is the mask
                const unsigned b = bits[u] >> (4 * (sub & 7));
                auto positive = [](unsigned bit, float x) { return !bit ? 0.f : x < 1.17549435e-38f ? 1.17549435e-38f : x; };
                v = make_float4(positive(b & 1u, v.x), positive(b & 2u, v.y), positive(b & 4u, v.z), positive(b & 8u, v.w));
            }
            unsigned word = 0;
            if (J.hmask) {                                // columns 8 m + 4 h + q: the nibbles of word h are the even or odd ones
                const unsigned lo = (unsigned)__shfl((int)bits[u], (int)(threadIdx.x & 48), 64), hi = (unsigned)__shfl((int)bits[u], (int)(threadIdx.x & 48) + 8, 64);
                const int h = sub & 1;
#pragma unroll
                for (int m = 0; m < 4; m++)
                    word |= ((lo >> (8 * m + 4 * h)) & 15u) << (4 * m) | ((hi >> (8 * m + 4 * h)) & 15u) << (16 + 4 * m);
            }
            if (r >= rows) continue;
            if (inside) *reinterpret_cast<float4*>(J.x + r * J.ld + col) = v;
            if (J.hmask && sub < 2) J.hmask[r * J.hld + J.hword + 2 * g + sub] = word;
        }
    }
}

// ------------------------------------------------------------------ linear
// What the backward keeps of the input, in one block: codes [N][kp] | scales [N][kp / 64] | sign bits [N][kp / 64][2 words]
// (x > 0), kp = K rounded up to 64.  Column c of a group is bit c & 31 of word c >> 5 for float32 and bit c >> 1 of word c & 1
// for the 16-bit types: a word is the lane mask of one tile of linear8_rows_kernel's result.
struct Keep { unsigned char* codes; float* scales; unsigned char* bits; int kp; };

static Keep carve_keep(char* base, long long N, int K, int what, size_t* bytes)
{
    Keep k = {};
    k.kp = (K + 63) / 64 * 64;
    char* p = base;
    if (what & GS4D_KEEP_CODES) {
        gs4d_obtain(p, k.codes, (size_t)N * k.kp);
        gs4d_obtain(p, k.scales, (size_t)N * (k.kp / 64));
    }
    if (what & GS4D_KEEP_SIGNS) gs4d_obtain(p, k.bits, (size_t)N * (k.kp / 8));
    if (bytes) *bytes = (size_t)(p - base) + 256;
    return k;
}

template <typename F> static int by_type(int dtype, F f)
{
    return dtype == GS4D_F32 ? f(float()) : dtype == GS4D_BF16 ? f(LbBf16()) : f(LbF16());
}
template <int V> struct Int { static constexpr int value = V; };
template <typename F> static int by_fmt(int fmt, F f)
{
    return fmt == GS4D_FMT_INT8 ? f(Int<GS4D_FMT_INT8>()) : fmt == GS4D_FMT_E4M3 ? f(Int<GS4D_FMT_E4M3>()) :
           fmt == GS4D_FMT_E5M2 ? f(Int<GS4D_FMT_E5M2>()) : f(Int<GS4D_FMT_UINT8>());
}

// What the matrix cores work on: 8 consecutive elements of a row per lane (lane & 31: the row of the operand, lane >> 5: which
// half of 16), as 16-bit numbers.  A float32 number is the sum of three bfloat16 numbers: itself rounded to nearest, what is left
// rounded to nearest, and what is left then (exact above 2^-100).  The second is below 2^-8 of the first and the third below 2^-17,
// each of either sign, and a product of two numbers is taken from the six largest of the nine term products: the three left out are
// below 2^-24 (1 + 2^-8) of it together, a rounding's worth.  (Terms cut off instead of rounded leave out up to 2^-21, always in one
// direction.)  A product within 2^-7 of the largest float32 number may become an infinity.  Six bfloat16 MFMAs against the float32
// one: 2.7 times its rate.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <typename T> constexpr int kTerms = 1;
template <> constexpr int kTerms<float> = 3;

template <typename T> __device__ __forceinline__ f32x16 mfma(const uint4& a, const uint4& b, const f32x16& c)
{
    if constexpr (__is_same(T, LbF16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// the upper halves of two words
__device__ __forceinline__ unsigned hi16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ float top8(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// two finite numbers -> their TERMS bfloat16 parts, packed.  ROUND: rounded to nearest (fits() says which numbers that is for), else
// the leading 8 bits each: of a sum of terms times ONE term all products are taken, and either is exact.
template <int TERMS, bool ROUND>
__device__ __forceinline__ void split2(float a, float b, unsigned (&o)[TERMS])
{
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
        if constexpr (ROUND) o[t] = __builtin_bit_cast(unsigned, __builtin_convertvector((lb_float2){a, b}, bf16x2));
        else o[t] = hi16(__float_as_uint(a), __float_as_uint(b));
        if (t + 1 < TERMS) {
            a -= ROUND ? __uint_as_float(o[t] << 16) : top8(a);
            b -= ROUND ? __uint_as_float(o[t] & 0xffff0000u) : top8(b);
        }
    }
}

template <int TERMS, bool ROUND>
__device__ __forceinline__ void split8(const float (&v)[8], uint4 (&o)[TERMS])
{
    unsigned w[4][TERMS];
#pragma unroll
    for (int q = 0; q < 4; q++) split2<TERMS, ROUND>(v[2 * q], v[2 * q + 1], w[q]);
#pragma unroll
    for (int t = 0; t < TERMS; t++) o[t] = make_uint4(w[0][t], w[1][t], w[2][t], w[3][t]);
}

// An infinity or a NaN of either operand of the float32 products.  Among three terms it would meet lower terms that are 0 and give a
// NaN where the product is an infinity.  So it is represented by its sign as a leading term, 1 or -1, and stands itself where it
// meets the other operand's leading term alone: a weight's as its third term, one of x in a product of its own (where there is one
// group of columns, its row is done again instead: AGAIN).  What the representatives add to the sum is finite and of no account beside
// an infinity; the sums of other rows and features come out the same.
// A number that would be rounded to an infinity has its leading 8 bits as a term beside the three of what is left.
__device__ __forceinline__ bool is_finite(unsigned bits) { return (bits & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ bool fits(unsigned bits) { return (bits & 0x7fffffffu) < 0x7f7f8000u; }
__device__ __forceinline__ float stand_in(unsigned bits)
{
    const float x = __uint_as_float(bits);
    const unsigned left = __float_as_uint(x - top8(x)), one = 0x3f800000u | (bits & 0x80000000u);
    const unsigned fit = (unsigned)((int)((bits & 0x7fffffffu) - 0x7f7f8000u) >> 31), fin = (unsigned)((int)((bits & 0x7fffffffu) - 0x7f800000u) >> 31);
    return __uint_as_float((bits & fit) | (((left & fin) | (one & ~fin)) & ~fit));       // masks: 32 of these as branches cost registers
}
// as bfloat16 numbers, 0 where there is nothing to represent
__device__ __forceinline__ unsigned special16(unsigned bits)
{
    const unsigned a = bits & 0x7fffffffu, fin = (unsigned)((int)(a - 0x7f800000u) >> 31), nan = (unsigned)((int)(0x7f800000u - a) >> 31);
    return ((bits >> 16) | (nan & 0x40u)) & ~fin;
}
__device__ __forceinline__ unsigned large16(unsigned bits)
{
    const unsigned a = bits & 0x7fffffffu, fit = (unsigned)((int)(a - 0x7f7f8000u) >> 31), fin = (unsigned)((int)(a - 0x7f800000u) >> 31);
    return (bits >> 16) & ~fit & fin;
}
template <typename F> __device__ __forceinline__ uint4 pack8(const unsigned (&e)[8], F f)
{
    return make_uint4(f(e[0]) | f(e[1]) << 16, f(e[2]) | f(e[3]) << 16, f(e[4]) | f(e[5]) << 16, f(e[6]) | f(e[7]) << 16);
}
__device__ __forceinline__ uint4 specials8(const unsigned (&e)[8]) { return pack8(e, [](unsigned b) { return special16(b); }); }
__device__ __forceinline__ uint4 larges8(const unsigned (&e)[8]) { return pack8(e, [](unsigned b) { return large16(b); }); }
// bfloat16 numbers with 0 in place of infinities and NaNs
__device__ __forceinline__ uint4 finite_only(const uint4& v)
{
    auto word = [](unsigned x) {
        if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
        if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
        return x;
    };
    return make_uint4(word(v.x), word(v.y), word(v.z), word(v.w));
}

// relu on the bits: a number with its sign bit set is a negative integer.  lowest = 0: relu, INT_MIN / -32768: nothing.
__device__ __forceinline__ unsigned relu_bits(unsigned x, int lowest) { return (unsigned)max((int)x, lowest); }
__device__ __forceinline__ unsigned relu_bits2(unsigned x, unsigned lowest2)
{
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(s16x2, x), __builtin_bit_cast(s16x2, lowest2)));
}
__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b)
{
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// A lane's share of a row's group of 64 columns: 4 steps of 8 elements, at columns 16 t + 8 h.
template <typename T> struct Group { uint4 w[4]; };
template <> struct Group<float> { uint4 w[8]; };

// VEC: C is a multiple of 8.  Columns past C are read somewhere inside the row (VEC) or with whatever follows the row; the caller
// clears them.  end: the end of the array, past which nothing is read (fix_end() reads the last row's last columns).
template <typename T, bool VEC>
__device__ __forceinline__ void load_group(Group<T>& g, const T* __restrict__ row, int c0, int C, const T* __restrict__ end)
{
    constexpr int PER = 16 / (int)sizeof(T);              // elements per 16 bytes
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const T* p = row + min(c0 + 16 * t, VEC ? C - 8 : C - 1);
        if (!VEC) p = p + 8 <= end ? p : reinterpret_cast<const T*>(kZeroPage);
#pragma unroll
        for (int q = 0; q < 8 / PER; q++) g.w[t * (8 / PER) + q] = load16(p + q * PER);
    }
}

// the columns that load_group() did not read because 8 of them would pass the end of the array
template <typename T>
__device__ __forceinline__ void fix_end(Group<T>& g, const T* __restrict__ row, int c0, int C, const T* __restrict__ end)
{
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int c = c0 + 16 * t;
        if (c >= C || row + c + 8 <= end) continue;
        unsigned e[8];
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if constexpr (sizeof(T) == 4) e[q] = __float_as_uint(row[min(c + q, C - 1)]);
            else e[q] = reinterpret_cast<const unsigned short*>(row)[min(c + q, C - 1)];
        }
        if constexpr (sizeof(T) == 4) {
            g.w[2 * t] = make_uint4(e[0], e[1], e[2], e[3]);
            g.w[2 * t + 1] = make_uint4(e[4], e[5], e[6], e[7]);
        } else {
            g.w[t] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }
}

template <typename T>
__device__ __forceinline__ void clear_past(Group<T>& g, int c0, int C)
{
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int left = C - c0 - 16 * t;                 // elements of this step inside the row
        if constexpr (sizeof(T) == 4) {
            unsigned* e = reinterpret_cast<unsigned*>(&g.w[2 * t]);
#pragma unroll
            for (int q = 0; q < 8; q++) e[q] = q < left ? e[q] : 0u;
        } else {
            unsigned* e = reinterpret_cast<unsigned*>(&g.w[t]);
#pragma unroll
            for (int q = 0; q < 4; q++) e[q] = 2 * q + 1 < left ? e[q] : 2 * q < left ? e[q] & 0xffffu : 0u;
        }
    }
}

// a NaN with its sign bit set would be rectified away
template <typename T>
__device__ __forceinline__ void positive_nans(Group<T>& g)
{
    unsigned* e = reinterpret_cast<unsigned*>(&g);
#pragma unroll
    for (int q = 0; q < (int)(sizeof(g) / 4); q++) {
        if constexpr (sizeof(T) == 4) {
            if ((e[q] & 0x7fffffffu) > 0x7f800000u) e[q] &= 0x7fffffffu;
        } else {
            constexpr unsigned kInf = __is_same(T, LbF16) ? 0x7c00u : 0x7f80u;
            if ((e[q] & 0x7fffu) > kInf) e[q] &= 0xffff7fffu;
            if ((e[q] >> 16 & 0x7fffu) > kInf) e[q] &= 0x7fffffffu;
        }
    }
}

// How the groups of the contraction and the column blocks are walked:
//   ROWS_ONE   one group, one column block (64 x 64 layers): nothing to prefetch within a tile, 16 waves of 128 registers
//              (100 k rows: 21 us)
//   ROWS_WIDE  one group, several column blocks: the group's operands stay in registers for all of them
//   ROWS_MANY  several groups: the next one is in flight while this one is multiplied, 8 waves (1.2 M x 256 -> 64: 476 to 496 us; 16
//              waves without the prefetch took 503 when this took 463)
//   ROWS_SPLIT several groups, few rows: the waves of a workgroup share a tile of rows, each takes groups of it, and the sums meet in
//              LDS (SPLIT)
enum { ROWS_ONE, ROWS_WIDE, ROWS_MANY, ROWS_SPLIT };
template <typename T, int NT, bool VEC, int MODE> constexpr int kRowsThreads = VEC && NT <= 2 && MODE == ROWS_ONE ? 1024 : 512;

struct RowsArgs {
    long long N; int C, F;                // rows, contraction length, features of the result
    const void* x; long long ldx;
    const void* w; long long wf, wc;      // element (feature f, contraction c) of the weight: w[f * wf + c * wc]
    const void* bias;
    void* y;                              // [N][F]
    int lowest;                           // relu_bits()
    Keep keep; int fmt;                   // forward: what to keep; dx: keep.bits masks the result
    int ncb, nwg, groups, chunk;          // sets of column blocks, workgroups per set, groups of 64 of the contraction, groups in LDS at once
    int blocks;                           // column blocks of NT * 32 features per set: 1, or more where the contraction is one group (ROWS_WIDE)
};

// Both products over the rows, y = x W^T (+ bias) and dx = dy W: a wave owns 32 rows and NT tiles of 32 features of
// v_mfma_f32_32x32x16; a lane streams its row from memory in groups of 64 columns and ends up with one feature of 16 rows, so
// that a row's results leave as whole lines.  (With features and rows exchanged a lane holds quads of one row, whose stores
// touch 32 lines each: the address units were busy 80 % of the time and the 1.2 M x 256 -> 64 product took 576 us.)  Tile nt
// holds the features 32 nt + lane, for 16-bit types the features 2 lane + (nt & 1) of 64, which leave as one word.
// The weight lies in LDS as MFMA operands, split once per workgroup, for as many groups as fit; the waves of a workgroup walk the
// rows.  What the backward needs of x is quantised on the way, from the registers that feed the product: x is read once.
template <typename T, int NT, bool VEC, bool DX, int MODE>
__global__ __launch_bounds__((kRowsThreads<T, NT, VEC, MODE>)) void linear8_rows_kernel(RowsArgs a)
{
    constexpr int TERMS = kTerms<T>, THREADS = kRowsThreads<T, NT, VEC, MODE>, WAVES = THREADS / 64, BLOCK = 4 * NT * TERMS * 64;
    constexpr bool SPLIT = MODE == ROWS_SPLIT;
    constexpr int PAIR = NT < 2 ? NT : 2;                 // tiles whose results leave together
    extern __shared__ uint4 s_w[];                        // [group][step][tile][term][lane], SPLIT: then [wave][tile of a pair][register][lane] of sums
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 31, h = lane >> 5;
    // workgroups that share rows differ by 8 in their number, i.e. run on one XCD behind one L2
    int cb, wg;
    if ((a.nwg & 7) == 0) {
        const int rest = blockIdx.x >> 3;
        cb = rest % a.ncb;
        wg = (rest / a.ncb) * 8 + (blockIdx.x & 7);
    } else {
        cb = blockIdx.x % a.ncb;
        wg = blockIdx.x / a.ncb;
    }
    const int C = a.C, F = a.F;
    int f0 = cb * a.blocks * NT * 32;
    const T* __restrict__ X = (const T*)a.x;
    const T* __restrict__ end = X + (a.N - 1) * a.ldx + C;
    const T* __restrict__ W = (const T*)a.w;
    auto feature = [&](int nt, int l) { return f0 + (sizeof(T) == 4 ? nt * 32 + l : (nt >> 1) * 64 + 2 * l + (nt & 1)); };
    auto stage = [&](int g0, int n, uint4* s_w) {         // groups g0 .. g0 + n - 1 of the weight, for the features from f0 on
        // U items at a time, their loads in flight together: one after the other, a 512 x 512 weight took 35 us to arrive
        constexpr int U = MODE == ROWS_MANY || SPLIT ? 4 : 1;     // (one group is few rounds, and the registers are worth more: 405 us, not 460)
        const int total = n * 4 * NT * 64;
        for (int e0 = tid; e0 < total; e0 += THREADS * U) {
            unsigned v[U][8];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int e = min(e0 + u * THREADS, total - 1);
                const int l = e & 63, nt = (e >> 6) % NT, step = (e >> 6) / NT;
                const int f = feature(nt, l & 31), c = g0 * 64 + step * 16 + 8 * (l >> 5);
                const T* p = W + (long long)min(f, F - 1) * a.wf;
                if (!DX && C >= 8) {                      // the row's columns, or its last 8
                    const T* w = p + min(c, C - 8);
                    if constexpr (sizeof(T) == 4) {
                        const uint4 x = load16(w), y = load16(w + 4);
                        v[u][0] = x.x; v[u][1] = x.y; v[u][2] = x.z; v[u][3] = x.w;
                        v[u][4] = y.x; v[u][5] = y.y; v[u][6] = y.z; v[u][7] = y.w;
                    } else {
                        const uint4 x = load16(w);
                        v[u][0] = x.x; v[u][1] = x.y; v[u][2] = x.z; v[u][3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        const T* w = p + (long long)min(c + q, C - 1) * a.wc;
                        if constexpr (sizeof(T) == 4) v[u][q] = __float_as_uint(*w);
                        else v[u][q] = *reinterpret_cast<const unsigned short*>(w);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int e = min(e0 + u * THREADS, total - 1);
                const int l = e & 63, nt = (e >> 6) % NT, step = (e >> 6) / NT;
                const int f = feature(nt, l & 31), c = g0 * 64 + step * 16 + 8 * (l >> 5);
                if (!DX && C >= 8 && c > C - 8) {         // columns past C - 8: read again, one by one
                    const T* p = W + (long long)min(f, F - 1) * a.wf;
                    unsigned t[8];
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        if constexpr (sizeof(T) == 4) t[q] = __float_as_uint(p[min(c + q, C - 1)]);
                        else t[q] = reinterpret_cast<const unsigned short*>(p)[min(c + q, C - 1)];
                    }
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        if constexpr (sizeof(T) == 4) v[u][q] = t[q];
                        else if (q < 4) v[u][q] = t[2 * q] | t[2 * q + 1] << 16;
                    }
                }
                if constexpr (sizeof(T) == 4) {
                    float x[8];
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        v[u][q] = f < F && c + q < C ? v[u][q] : 0u;
                        x[q] = __uint_as_float(v[u][q]);
                    }
                    uint4 o[TERMS];
                    split8<TERMS, true>(x, o);
                    const unsigned top2 = max_u16x2(max_u16x2(o[0].x & 0x7fff7fffu, o[0].y & 0x7fff7fffu), max_u16x2(o[0].z & 0x7fff7fffu, o[0].w & 0x7fff7fffu));
                    if (max(top2 & 0xffffu, top2 >> 16) >= 0x7f80u) {      // not all fits(): a weight has no term to spare: its leading bits and two terms of what is left
                        auto join = [](const uint4& a, const uint4& b) { return make_uint4(a.x | b.x, a.y | b.y, a.z | b.z, a.w | b.w); };
                        auto first = [](unsigned b) {     // (what rounding gives, but for numbers that do not fit)
                            const float x = __uint_as_float(b);
                            return fits(b) ? (unsigned)__builtin_bit_cast(unsigned short, (__bf16)x) : is_finite(b) ? b >> 16 : 0x3f80u | b >> 31 << 15;
                        };
                        uint4 two[2];
#pragma unroll
                        for (int q = 0; q < 8; q++) x[q] = is_finite(v[u][q]) ? x[q] - __uint_as_float(first(v[u][q]) << 16) : 0.f;
                        split8<2, true>(x, two);
                        o[0] = pack8(v[u], first);
                        o[1] = two[0];
                        o[TERMS - 1] = join(two[1], specials8(v[u]));
                    }
#pragma unroll
                    for (int t = 0; t < TERMS; t++) s_w[((step * NT + nt) * TERMS + t) * 64 + l] = o[t];
                } else {
                    unsigned x[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        x[q] = !DX && C >= 8 ? v[u][q] : v[u][2 * q] | v[u][2 * q + 1] << 16;
                        x[q] = f >= F || c + 2 * q >= C ? 0u : c + 2 * q + 1 < C ? x[q] : x[q] & 0xffffu;
                    }
                    s_w[(step * NT + nt) * 64 + l] = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
        }
    };
    const int ntile = (int)((a.N + 31) >> 5);
    const bool keeping = !DX && cb == 0 && (a.keep.codes || a.keep.bits);
    auto row_of = [&](long long tile) { const long long r = tile * 32 + j; return X + (r < a.N ? r : a.N - 1) * a.ldx; };
    long long tile = SPLIT ? wg : (long long)wave * a.nwg + wg;
    constexpr int TILES = SPLIT ? 1 : WAVES;              // per workgroup and round
    // one group of columns, float32: rows whose numbers are not all fits() are done again at the end, one by one, where registers are
    // free (taken care of among the others they cost a 64 -> 64 input gradient of 100 k rows 28 us instead of 18); bit i: in the rounds i modulo 64
    constexpr bool AGAIN = TERMS > 1 && (MODE == ROWS_ONE || MODE == ROWS_WIDE);
    unsigned long long again = 0;
    const long long tile0 = tile;
    Group<T> cur;
    // the waves start at different groups: a row of several 256-byte groups, read by all waves in step, would keep to a fraction of
    // the memory channels at a time
    const int turn = SPLIT ? wave : a.chunk >= a.groups ? wave % a.groups : 0;
    auto group_at = [&](int gi) { const int g = gi + turn; return SPLIT || g < a.groups ? g : g - a.groups; };
    load_group<T, VEC>(cur, row_of(tile), turn * 64 + 8 * h, C, end);      // in flight while the weight is staged
    if constexpr (MODE == ROWS_WIDE) {
        for (int k = 0; k < a.blocks; k++) { stage(0, 1, s_w + k * BLOCK); f0 += NT * 32; }
        f0 -= a.blocks * NT * 32;
    } else if (a.chunk >= a.groups) {
        stage(0, a.groups, s_w);
    }
    __syncthreads();
    for (long long base = 0; base * a.nwg < ntile; base += TILES, tile += (long long)TILES * a.nwg) {      // uniform: every wave takes part in the barriers
        const long long row = tile * 32 + j;
        const bool live = row < a.N;
        f32x16 acc[NT];
        unsigned sign[NT];                                // dx: the sign bits of the lane's row for the tiles' features
        auto begin = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float b = !SPLIT && !DX && a.bias ? lb_load(((const T*)a.bias)[min(feature(nt, j), F - 1)]) : 0.f;
#pragma unroll
                for (int r = 0; r < 16; r++) acc[nt][r] = b;
            }
            if (DX && a.keep.bits) {
                const unsigned* p = reinterpret_cast<const unsigned*>(a.keep.bits) + (live ? row : a.N - 1) * (a.keep.kp / 32);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) sign[nt] = p[min((f0 >> 5) + nt, a.keep.kp / 32 - 1)];
            }
        };
        auto step = [&](const uint4 (&xs)[TERMS], const uint4* __restrict__ wl) {
            uint4 ws[NT][TERMS];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int u = 0; u < TERMS; u++) ws[nt][u] = wl[(nt * TERMS + u) * 64];
#pragma unroll
            for (int u = TERMS - 1; u >= 0; u--)          // the smallest products first
#pragma unroll
                for (int z = 0; z <= u; z++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) acc[nt] = mfma<T>(xs[u - z], ws[nt][z], acc[nt]);
        };
        // what stand_in() leaves out of a step
        auto add_specials = [&](const unsigned (&e)[8], const uint4* __restrict__ wl) {
            const uint4 sp = specials8(e), lg = larges8(e);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                __builtin_amdgcn_sched_barrier(0);        // rare: few registers count, not time
                acc[nt] = mfma<T>(sp, wl[nt * TERMS * 64], acc[nt]);
#pragma unroll
                for (int u = TERMS - 1; u >= 0; u--) {
                    __builtin_amdgcn_sched_barrier(0);
                    acc[nt] = mfma<T>(lg, finite_only(wl[(nt * TERMS + u) * 64]), acc[nt]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        // register r is the row rr + 4 h of the tile, rr = (r & 3) + 8 (r >> 2); o: its results of the tiles nt, nt + 1
        auto put = [&](T* __restrict__ yt, bool whole, int rr, int nt, const float (&o)[PAIR]) {
            if (!whole && tile * 32 + rr + 4 * h >= a.N) return;
            T* __restrict__ y = yt + (long long)rr * F + feature(nt, j);
            if constexpr (sizeof(T) == 2) {
                const T two[2] = {lb_store<T>(o[0]), lb_store<T>(o[1])};
                if (feature(nt, j) + 1 < F) __builtin_memcpy(y, two, 4);
                else if (feature(nt, j) < F) *y = two[0];
            } else {
#pragma unroll
                for (int u = 0; u < PAIR; u++)
                    if (feature(nt + u, j) < F) y[32 * u] = o[u];
            }
        };
        auto finish = [&]() {
            const bool whole = tile * 32 + 32 <= a.N;
            T* __restrict__ yt = (T*)a.y + (tile * 32 + 4 * h) * F;
#pragma unroll
            for (int r = 0; r < 16; r++)
#pragma unroll
                for (int nt = 0; nt < NT; nt += PAIR) {
                    float o[PAIR];
#pragma unroll
                    for (int u = 0; u < PAIR; u++) {
                        o[u] = acc[nt + u][r];
                        if (DX && a.keep.bits) {
                            const int rr = (r & 3) + 8 * (r >> 2);
                            const unsigned long long lanes = (unsigned long long)(unsigned)__builtin_amdgcn_readlane(sign[nt + u], rr + 4) << 32 | (unsigned)__builtin_amdgcn_readlane(sign[nt + u], rr);
                            o[u] = __builtin_amdgcn_inverse_ballot_w64(lanes) ? o[u] : 0.f;
                        }
                    }
                    put(yt, whole, (r & 3) + 8 * (r >> 2), nt, o);
                }
        };
        // the waves' sums of a pair of tiles side by side in LDS, then two of the 16 registers per wave
        auto join = [&]() {
            const bool whole = tile * 32 + 32 <= a.N;
            T* __restrict__ yt = (T*)a.y + (tile * 32 + 4 * h) * F;
            float* __restrict__ part = reinterpret_cast<float*>(s_w + (size_t)a.groups * BLOCK);
            const int parts = min(a.groups, WAVES);
#pragma unroll
            for (int nt = 0; nt < NT; nt += PAIR) {
                if (wave < parts) {
#pragma unroll
                    for (int u = 0; u < PAIR; u++)
#pragma unroll
                        for (int r = 0; r < 16; r++) part[((wave * PAIR + u) * 16 + r) * 64 + lane] = acc[nt + u][r];
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < 16 / WAVES; k++) {
                    const int r = wave * (16 / WAVES) + k, rr = (r & 3) + 8 * (r >> 2);
                    float o[PAIR];
#pragma unroll
                    for (int u = 0; u < PAIR; u++) {
                        o[u] = !DX && a.bias ? lb_load(((const T*)a.bias)[min(feature(nt + u, j), F - 1)]) : 0.f;
                        for (int q = 0; q < parts; q++) o[u] += part[((q * PAIR + u) * 16 + r) * 64 + lane];
                        if (DX && a.keep.bits) o[u] = (unsigned)__shfl((int)sign[nt + u], rr + 4 * h, 64) >> j & 1u ? o[u] : 0.f;
                    }
                    put(yt, whole, rr, nt, o);
                }
                __syncthreads();
            }
        };
        if (MODE != ROWS_WIDE) begin();
        for (int gi = 0; gi < (SPLIT ? a.groups - wave : a.groups); gi += SPLIT ? WAVES : 1) {
            const int g = group_at(gi);
            int Cn = a.C;
            asm("" : "+s"(Cn));                           // column limits are recomputed: kept over the loop they would spill
            // (ROWS_WIDE has one group and does not take this, but the compiler's order of its code is worse without: 1.2 M x 64 -> 256
            // 453 us, not 399)
            if (!SPLIT && MODE != ROWS_ONE && a.chunk < a.groups && gi % a.chunk == 0) {
                __syncthreads();
                stage(gi, min(a.chunk, a.groups - gi), s_w);
                __syncthreads();
            }
            if (g * 64 + 64 > Cn) {
                if (!VEC) fix_end(cur, row_of(tile), g * 64 + 8 * h, Cn, end);
                clear_past(cur, g * 64 + 8 * h, Cn);
            }
            const uint4* __restrict__ wl = s_w + (size_t)(MODE == ROWS_MANY && a.chunk < a.groups ? gi % a.chunk : g) * 4 * NT * TERMS * 64 + lane;
            constexpr int NEXT = SPLIT ? WAVES : 1;
            const bool more = SPLIT ? g + NEXT < a.groups : gi + 1 < a.groups;
            Group<T> nxt;
            if (MODE == ROWS_MANY || SPLIT) load_group<T, VEC>(nxt, row_of(more ? tile : tile + (long long)TILES * a.nwg), group_at(more ? gi + NEXT : 0) * 64 + 8 * h, Cn, end);
            // the group's largest number (of the kept values) and whether anything in it is no finite number
            unsigned m = 0, odd = 0;
            float v[4][8];
            if constexpr (sizeof(T) == 4 && DX) {         // (nothing else needs the magnitudes here; a NaN needs no care)
                float most = 0.f;
                const float* e = reinterpret_cast<const float*>(&cur);
#pragma unroll
                for (int q = 0; q < 32; q += 2) asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(most) : "v"(e[q]), "v"(e[q + 1]));
                odd = !(most < __uint_as_float(0x7f7f8000u));
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int t = 0; t < 8; t++) odd = max(max(odd, max(cur.w[t].x & 0x7fffffffu, cur.w[t].y & 0x7fffffffu)), max(cur.w[t].z & 0x7fffffffu, cur.w[t].w & 0x7fffffffu));
                odd = odd >= 0x7f7f8000u;                 // !fits()
            } else {
                unsigned o2 = 0;
#pragma unroll
                for (int t = 0; t < 4; t++) o2 = max_u16x2(max_u16x2(o2, max_u16x2(cur.w[t].x & 0x7fff7fffu, cur.w[t].y & 0x7fff7fffu)), max_u16x2(cur.w[t].z & 0x7fff7fffu, cur.w[t].w & 0x7fff7fffu));
                odd = max(o2 & 0xffffu, o2 >> 16) >= (__is_same(T, LbF16) ? 0x7c00u : 0x7f80u);
            }
            const bool any = __builtin_amdgcn_ballot_w64(odd) != 0;
            if (!DX && any) positive_nans(cur);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const unsigned* e = reinterpret_cast<const unsigned*>(&cur.w[2 * t]);
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        const unsigned r = DX ? e[q] : relu_bits(e[q], a.lowest);
                        m = max(m, r & 0x7fffffffu);
                        v[t][q] = __uint_as_float(r);
                    }
                }
            } else if constexpr (!DX) {
                const unsigned low2 = a.lowest ? 0x80008000u : 0u;
                unsigned m2 = 0;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    unsigned* e = reinterpret_cast<unsigned*>(&cur.w[t]);
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        e[q] = relu_bits2(e[q], low2);
                        m2 = max_u16x2(m2, e[q] & 0x7fff7fffu);
                    }
                }
                m = __float_as_uint(low16<T>(max(m2 & 0xffffu, m2 >> 16)));
            }
            if (keeping) {
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const unsigned* e = reinterpret_cast<const unsigned*>(&cur.w[t]);
#pragma unroll
                        for (int q = 0; q < 4; q++) { v[t][2 * q] = low16<T>(e[q]); v[t][2 * q + 1] = high16<T>(e[q]); }
                    }
                }
                if (a.keep.bits) {                        // relu: every number is at least 0 here
                    unsigned w[2] = {0, 0};
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            const unsigned positive = min(__float_as_uint(v[t][q]), 1u);
                            if (sizeof(T) == 4) w[t >> 1] |= positive << (16 * (t & 1) + q);
                            else w[q & 1] |= positive << (8 * t + (q >> 1));
                        }
                    const int at = sizeof(T) == 4 ? 8 * h : 4 * h;
                    w[0] <<= at;
                    w[1] <<= at;
                    w[0] |= (unsigned)__shfl_xor((int)w[0], 32, 64);
                    w[1] |= (unsigned)__shfl_xor((int)w[1], 32, 64);
                    if (live && h == 0) *reinterpret_cast<uint2*>(a.keep.bits + (size_t)row * (a.keep.kp / 8) + g * 8) = make_uint2(w[0], w[1]);
                }
                if (a.keep.codes) {
                    m = max(m, (unsigned)__shfl_xor((int)m, 32, 64));
                    unsigned char* code = a.keep.codes + (size_t)row * a.keep.kp + g * 64 + 16 * h;
                    auto encode = [&](auto f) {
                        constexpr int FMT = decltype(f)::value;
                        const LbScale sc = lb_scale<FMT>(m);
#pragma unroll
                        for (int t = 0; t < 4; t += 2) {
                            unsigned w[4];
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const float* p = &v[t + (q >> 1)][4 * (q & 1)];
                                w[q] = lb_encode4<FMT>(p[0] * sc.inv, p[1] * sc.inv, p[2] * sc.inv, p[3] * sc.inv);
                            }
                            // the halves swap, so that a lane has 16 codes in a row: step t for h = 0, step t + 1 for h = 1
                            const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                            if (live) *reinterpret_cast<uint4*>(code + 16 * t) = make_uint4(x[0], y[0], x[1], y[1]);
                        }
                        if (live && h == 0) a.keep.scales[(size_t)row * (a.keep.kp / 64) + g] = sc.s;
                    };
                    if (a.fmt == GS4D_FMT_INT8) encode(Int<GS4D_FMT_INT8>());
                    else if (a.fmt == GS4D_FMT_UINT8) encode(Int<GS4D_FMT_UINT8>());
                    else if (a.fmt == GS4D_FMT_E4M3) encode(Int<GS4D_FMT_E4M3>());
                    else encode(Int<GS4D_FMT_E5M2>());
                }
            }
            if constexpr (AGAIN) {
                again |= (unsigned long long)any << (base / TILES & 63);
            } else if constexpr (TERMS > 1) {
                if (any) {
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        unsigned e[8];
#pragma unroll
                        for (int q = 0; q < 8; q++) e[q] = __float_as_uint(v[t][q]);
                        add_specials(e, wl + t * NT * TERMS * 64);
#pragma unroll
                        for (int q = 0; q < 8; q++) v[t][q] = stand_in(e[q]);
                    }
                }
            }
            if constexpr (MODE == ROWS_WIDE) {
                // one group: its operands stay in registers for all of the workgroup's features
                uint4 xs[4][TERMS];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    if constexpr (sizeof(T) == 4) split8<TERMS, true>(v[t], xs[t]);
                    else xs[t][0] = cur.w[t];
                }
#pragma unroll 1
                for (int k = 0; k < a.blocks; k++) {
                    begin();
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        step(xs[t], s_w + k * BLOCK + t * NT * TERMS * 64 + lane);
                    }
                    finish();
                    f0 += NT * 32;
                }
                f0 -= a.blocks * NT * 32;
                __builtin_amdgcn_sched_barrier(0);
                load_group<T, VEC>(cur, row_of(tile + (long long)WAVES * a.nwg), 8 * h, Cn, end);
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    if (MODE == ROWS_ONE) __builtin_amdgcn_sched_barrier(0);      // a step at a time: hoisted splits and weights would spill
                    uint4 xs[TERMS];
                    if constexpr (sizeof(T) == 4) split8<TERMS, true>(v[t], xs);
                    else xs[0] = cur.w[t];
                    step(xs, wl + t * NT * TERMS * 64);
                }
                if (MODE == ROWS_MANY || SPLIT) {
                    cur = nxt;
                } else {
                    __builtin_amdgcn_sched_barrier(0);
                    load_group<T, VEC>(cur, row_of(tile + (long long)WAVES * a.nwg), 8 * h, Cn, end);
                }
            }
        }
        if constexpr (SPLIT) join();
        else if (MODE != ROWS_WIDE) finish();
    }
    if constexpr (AGAIN) {
        if (!again) return;
        __threadfence();                                  // the wave stores to the same places again
        const int f1 = min(F, f0 + a.blocks * NT * 32);
        long long round = 0;
        for (long long t = tile0; t < ntile; t += (long long)TILES * a.nwg, round++) {
            if (!(again >> (round & 63) & 1)) continue;
            for (long long row = t * 32; row < t * 32 + 32 && row < a.N; row++) {
                unsigned e = lane < C ? __float_as_uint(reinterpret_cast<const float*>(X)[row * a.ldx + lane]) : 0u;
                if (!__builtin_amdgcn_ballot_w64(!fits(e))) continue;
                if (!DX && (e & 0x7fffffffu) <= 0x7f800000u) e = relu_bits(e, a.lowest);      // (a NaN of either sign stays one)
                for (int fb = f0; fb < f1; fb += 64) {
                    const int f = min(fb + lane, f1 - 1);
                    const float* __restrict__ w = reinterpret_cast<const float*>(W) + (long long)f * a.wf;
                    float sum = !DX && a.bias ? reinterpret_cast<const float*>(a.bias)[f] : 0.f;
                    for (int c = 0; c < C; c++) sum = fmaf(__uint_as_float((unsigned)__builtin_amdgcn_readlane((int)e, c)), w[(long long)c * a.wc], sum);
                    if (DX && a.keep.bits && !(reinterpret_cast<const unsigned*>(a.keep.bits)[row * (a.keep.kp / 32) + (f >> 5)] >> (f & 31) & 1u)) sum = 0.f;
                    if (fb + lane < f1) reinterpret_cast<float*>(a.y)[row * F + f] = sum;
                }
            }
        }
    }
}

// A few rows (a single query): 16 lanes per feature read its weights once, 4 columns each, and multiply them with
// all the rows.  No staging, so the latency is one round trip to memory (one row of 64 -> 64: 2.5 us, with the matrix cores 10).
// These kernels take 1 us per 7 M products forward and per 15 M backward (per 5 M and 6 M where the weight is read from memory), the
// others first stage and split the weight, which takes 0.08 us (forward float32; 16 bits 0.03, backward 0.055 and 0.037) per column of
// the contraction however few the rows, and then go as many rows at once: hence the first rule of each line for the row count and
// the second for weights so large that the rows, times the features, are read or multiplied longer than that.  Measured, these
// against those, in us: float32 forward 64 rows of 2048 -> 1024 25 : 156, 2048 of 64 -> 512 20 : 19, 4096 of 64 -> 512 37 : 21, 64 of
// 16384 -> 16384 3869 : 1263; backward 1024 of 512 -> 512 19 : 33, 2048 33 : 32, 64 of 16384 -> 16384 2794 : 898.  16-bit forward 256 of
// 512 -> 512 13 : 18, 1024 of 64 -> 512 11 : 15, 2048 20 : 16, 200 of 2048 -> 1024 63 : 61, 64 of 16384 -> 16384 3370 : 542; backward 2048
// of 512 -> 64 8 : 19, 512 of 2048 -> 1024 71 : 40, 64 of 16384 -> 16384 2358 : 610.
#define FEW_ROWS 4            // per workgroup
static bool few(int dtype, bool dx, long long N, int K, int M)
{
    const bool f32 = dtype == GS4D_F32;
    if (dx) return N <= 4096 && (N - 200) * K * M <= 1ll << (f32 ? 28 : 27) && N * K <= (f32 ? 350000 : 120000) + (1ll << 28) / M;
    return f32 ? N <= 4096 && (N - 500) * K * M <= 1ll << 26 && N * M <= 400000 + (1ll << 26) / K
               : N <= 2048 && (N - 200) * K * M <= 1ll << 25 && N * M <= 130000 + (1ll << 25) / K;
}
template <typename T>
__global__ __launch_bounds__(256) void linear8_few_kernel(RowsArgs a)
{
    const int fblocks = (a.F + 15) / 16;
    if ((int)blockIdx.x >= fblocks) {
        const int ng = a.keep.kp / 64, here = min(FEW_ROWS, (int)a.N - (int)blockIdx.y * FEW_ROWS);
        const int item = min(((int)blockIdx.x - fblocks) * 16 + (int)(threadIdx.x >> 4), here * ng - 1), row = blockIdx.y * FEW_ROWS + item / ng, g = item % ng, sub = threadIdx.x & 15,
                  col = g * 64 + 4 * sub;
        const T* __restrict__ x = (const T*)a.x + row * a.ldx;
        float e[4];
        unsigned m = 0, w0 = 0, w1 = 0;                   // the sign words: column c of the group is bit c & 31 of word c >> 5, or
#pragma unroll                                            // bit c >> 1 of word c & 1 (16-bit types)
        for (int q = 0; q < 4; q++) {
            e[q] = col + q < a.C ? lb_load(x[min(col + q, a.C - 1)]) : 0.f;
            if (!a.lowest && e[q] < 0.f) e[q] = 0.f;
            m = max(m, lb_abs_bits(e[q]));
            const unsigned positive = lb_abs_bits(e[q]) ? 1u : 0u;
            const int c = 4 * sub + q;
            if (sizeof(T) == 4) { if (c < 32) w0 |= positive << (c & 31); else w1 |= positive << (c & 31); }
            else if (q & 1) w1 |= positive << (c >> 1);
            else w0 |= positive << (c >> 1);
        }
        m = group_max(m, 4);
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) { w0 |= (unsigned)__shfl_xor((int)w0, k, 64); w1 |= (unsigned)__shfl_xor((int)w1, k, 64); }
        if (a.keep.bits && sub == 0) *reinterpret_cast<uint2*>(a.keep.bits + (size_t)row * (a.keep.kp / 8) + g * 8) = make_uint2(w0, w1);
        auto encode = [&](auto fm) {
            constexpr int FMT = decltype(fm)::value;
            const LbScale sc = lb_scale<FMT>(m);
            *reinterpret_cast<unsigned*>(a.keep.codes + (size_t)row * a.keep.kp + col) = lb_encode4<FMT>(e[0] * sc.inv, e[1] * sc.inv, e[2] * sc.inv, e[3] * sc.inv);
            if (sub == 0) a.keep.scales[(size_t)row * ng + g] = sc.s;
        };
        if (!a.keep.codes) return;
        if (a.fmt == GS4D_FMT_INT8) encode(Int<GS4D_FMT_INT8>());
        else if (a.fmt == GS4D_FMT_UINT8) encode(Int<GS4D_FMT_UINT8>());
        else if (a.fmt == GS4D_FMT_E4M3) encode(Int<GS4D_FMT_E4M3>());
        else encode(Int<GS4D_FMT_E5M2>());
        return;
    }
    const int sub = threadIdx.x & 15, f = blockIdx.x * 16 + (threadIdx.x >> 4), fc = min(f, a.F - 1), C = a.C;
    const T* __restrict__ w = (const T*)a.w + (long long)fc * a.wf;
    const T* __restrict__ x = (const T*)a.x;
    const float floor = a.lowest ? -INFINITY : 0.f;
    const int r0 = blockIdx.y * FEW_ROWS, last = (int)a.N - 1;
    float acc[FEW_ROWS] = {};
    for (int c = 4 * sub; c < C; c += 64) {
        float wv[4], xv[FEW_ROWS][4];
        if (c + 4 <= C) {
            T e[4], g[FEW_ROWS][4];
            __builtin_memcpy(e, w + c, sizeof(e));
#pragma unroll
            for (int r = 0; r < FEW_ROWS; r++) __builtin_memcpy(g[r], x + min(r0 + r, last) * a.ldx + c, sizeof(e));
#pragma unroll
            for (int q = 0; q < 4; q++) {
                wv[q] = lb_load(e[q]);
#pragma unroll
                for (int r = 0; r < FEW_ROWS; r++) xv[r][q] = lb_load(g[r][q]);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int k = min(c + q, C - 1);
                wv[q] = c + q < C ? lb_load(w[k]) : 0.f;
#pragma unroll
                for (int r = 0; r < FEW_ROWS; r++) xv[r][q] = c + q < C ? lb_load(x[min(r0 + r, last) * a.ldx + k]) : 0.f;
            }
        }
#pragma unroll
        for (int r = 0; r < FEW_ROWS; r++)
#pragma unroll
            for (int q = 0; q < 4; q++) acc[r] = fmaf(xv[r][q] < floor ? floor : xv[r][q], wv[q], acc[r]);      // a NaN stays one
    }
    const float b = a.bias ? lb_load(((const T*)a.bias)[fc]) : 0.f;
#pragma unroll
    for (int r = 0; r < FEW_ROWS; r++) {
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) acc[r] += __shfl_xor(acc[r], k, 64);
        if (sub == 0 && f < a.F && r0 + r <= last) ((T*)a.y)[(long long)(r0 + r) * a.F + f] = lb_store<T>(acc[r] + b);
    }
}

// dx of a few rows: a workgroup takes 64 columns, 4 per lane, and deals the rows of the weight to 16 slices, summed through LDS
template <typename T>
__global__ __launch_bounds__(256) void linear8_few_dx_kernel(RowsArgs a)
{
    __shared__ float s_part[16][FEW_ROWS][64];
    const int sub = threadIdx.x & 15, slice = threadIdx.x >> 4, k = blockIdx.x * 64 + 4 * sub, F = a.F, C = a.C;
    const int r0 = blockIdx.y * FEW_ROWS, last = (int)a.N - 1;
    const T* __restrict__ w = (const T*)a.w;
    const T* __restrict__ dy = (const T*)a.x;
    float acc[FEW_ROWS][4] = {};
#pragma unroll 4
    for (int m = slice; m < C; m += 16) {
        float wv[4];
        if (k + 4 <= F) {
            T e[4];
            __builtin_memcpy(e, w + (long long)m * F + k, sizeof(e));
#pragma unroll
            for (int q = 0; q < 4; q++) wv[q] = lb_load(e[q]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++) wv[q] = lb_load(w[(long long)m * F + min(k + q, F - 1)]);
        }
#pragma unroll
        for (int r = 0; r < FEW_ROWS; r++) {
            const float d = lb_load(dy[(long long)min(r0 + r, last) * a.ldx + m]);
#pragma unroll
            for (int q = 0; q < 4; q++) acc[r][q] = fmaf(d, wv[q], acc[r][q]);
        }
    }
#pragma unroll
    for (int r = 0; r < FEW_ROWS; r++)
#pragma unroll
        for (int q = 0; q < 4; q++) s_part[slice][r][4 * sub + q] = acc[r][q];
    __syncthreads();
    const int r = threadIdx.x >> 6, c = threadIdx.x & 63, row = r0 + r, col = blockIdx.x * 64 + c;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 16; q++) v += s_part[q][r][c];
    if (row > last || col >= F) return;
    if (a.keep.bits) {
        const unsigned* bits = reinterpret_cast<const unsigned*>(a.keep.bits) + (size_t)row * (a.keep.kp / 32) + 2 * blockIdx.x;
        if (!(sizeof(T) == 4 ? bits[c >> 5] >> (c & 31) & 1u : bits[c & 1] >> (c >> 1) & 1u)) v = 0.f;
    }
    ((T*)a.y)[(long long)row * F + col] = lb_store<T>(v);
}

// dW[m][k] = sum over rows r of dy[r][m] s[r] c[r][k] with the kept codes c and their group's scale s.  The contraction runs over
// the ROWS, and any 8 rows may be the 8 elements a lane supplies as long as both operands agree: a lane loads column pairs
// (2 i, 2 i + 1) of dy and of the codes straight from memory, row after row, coalesced, and no transposition through LDS is needed.
// Tile t of the result then holds the columns 2 i + t.  The codes are exact in bfloat16 (8 significant bits), so the rounding
// lies in dy s alone, a float32 number, whose 24 bits are three bfloat16 numbers, for every type of dy.
// A workgroup: 64 columns m, GW groups of 64 columns k (a wave each) and 8 / GW row slices per group, summed through LDS;
// one slab of partial sums per workgroup.  Bound by the vector instructions that form and split dy s, once per group of columns:
// 180 of them and 12 MFMAs a step of 16 rows (float32, int8).  1.2 M x 256 -> 64: 238 to 244 us (reading once: 135), 65536 x 512 -> 512
// fp16 142 to 148 us (two terms of dy s, which lose up to 2^-15 of a product, 116 to 126), 100 k x 64 -> 64 13 us.
struct DwArgs {
    long long N; int K, M;
    const void* dy; Keep keep;
    long long per;                        // rows per chunk
    int gw, groups, mtiles, chunks;
    float* slabs;                         // [chunk][m tile][group][64 registers][64 lanes], then [chunk][m tile][64] of db
};

// lane Q of the lane's 16
template <int Q> __device__ __forceinline__ float row_lane(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + Q, 0xF, 0xF, true));
}

template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(512) void linear8_dw_kernel(DwArgs a)
{
    constexpr int TERMS = 3;
    __shared__ float s_red[4][64 * 64];
    __shared__ float s_db[8][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 31, h = lane >> 5;
    const int chunk = blockIdx.x % a.chunks, rest = blockIdx.x / a.chunks, mt = rest % a.mtiles, z = rest / a.mtiles;
    const int g = z * a.gw + wave % a.gw, slice = wave / a.gw, slices = 8 / a.gw;
    const long long n0 = chunk * a.per, n1 = n0 + a.per < a.N ? n0 + a.per : a.N;
    const bool mine = g < a.groups;
    const int gc = min(g, a.groups - 1), m = mt * 64 + 2 * i, kp = a.keep.kp, ng = kp / 64, M = a.M;
    const T* __restrict__ dy = (const T*)a.dy;
    // VEC: two columns at once, at any alignment; an odd M's last column is the second of its pair
    const int mc = VEC ? min(m, M - 2) : 0;
    const bool shifted = VEC && m == M - 1;
    const unsigned char* __restrict__ codes = a.keep.codes + gc * 64;
    const float* __restrict__ scales = a.keep.scales + gc;
    // a load's address is the wave's row plus the lane's share, which does not change
    const unsigned dlane = (unsigned)((8 * h * M + mc) * (int)sizeof(T)), clane = (unsigned)(8 * h * kp + 2 * i);
    struct Rows { unsigned d[8][sizeof(T) / 2]; unsigned short c[8]; float s; };
    // rows r0 + 8 h + q; LAST: some of them may lie past the end
    auto load = [&](Rows& r, long long r0, auto last) {
        constexpr bool LAST = decltype(last)::value != 0;
        unsigned dl = dlane, cl = clane;
        asm("" : "+v"(dl), "+v"(cl));                     // no address kept over the loop: the row's part stays scalar, the lane's 32 bits
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const char* pd = reinterpret_cast<const char*>(dy + (r0 + q) * M);
            const char* pc = reinterpret_cast<const char*>(codes + (r0 + q) * kp);
            pd += dl;
            pc += cl;
            if (LAST && r0 + 8 * h + q >= a.N) {          // the last row instead
                pd = reinterpret_cast<const char*>(dy + (a.N - 1) * M + mc);
                pc = reinterpret_cast<const char*>(codes + (a.N - 1) * kp + 2 * i);
            }
            const T* p = reinterpret_cast<const T*>(pd);
            if constexpr (sizeof(T) == 4) {
                if constexpr (VEC) __builtin_memcpy(r.d[q], p, 8);
                else r.d[q][0] = r.d[q][1] = __float_as_uint(p[0]);
            } else {
                if constexpr (VEC) __builtin_memcpy(r.d[q], p, 4);
                else r.d[q][0] = *reinterpret_cast<const unsigned short*>(p);
            }
            r.c[q] = *reinterpret_cast<const unsigned short*>(pc);
        }
        // lane q of 16 has the scale of row r0 + 8 h + q (q < 8), broadcast where it is used.  (As scalar loads, which return in any
        // order, they made each step wait for the loads of the next: 1.2 M x 256 -> 64 292 us.)
        const long long n = r0 + 8 * h + (lane & 7);
        r.s = scales[(LAST && n >= a.N ? a.N - 1 : n) * ng];
        if (LAST && n >= n1) r.s = 0.f;
    };
    f32x16 acc[2][2] = {};
    float db0 = 0.f, db1 = 0.f;
    int turn = wave % a.gw;
    auto add = [&](const Rows& cur, long long r0, auto last, auto any) {
        constexpr bool LAST = decltype(last)::value != 0, ANY = decltype(any)::value != 0;
        float d0[8], d1[8], c0[8], c1[8];
        const float sq[8] = {row_lane<0>(cur.s), row_lane<1>(cur.s), row_lane<2>(cur.s), row_lane<3>(cur.s),
                             row_lane<4>(cur.s), row_lane<5>(cur.s), row_lane<6>(cur.s), row_lane<7>(cur.s)};
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if constexpr (sizeof(T) == 4) { d0[q] = __uint_as_float(cur.d[q][0]); d1[q] = __uint_as_float(cur.d[q][1]); }
            else { d0[q] = low16<T>(cur.d[q][0]); d1[q] = high16<T>(cur.d[q][0]); }
            if (VEC) d0[q] = shifted ? d1[q] : d0[q];
            if (LAST && r0 + 8 * h + q >= n1) { d0[q] = 0.f; d1[q] = 0.f; }
        }
        // the groups' waves of a slice take turns at the column sums of dy
        if (turn == 0) {
            asm volatile("");                             // a branch: as selects the sums would be formed by all
#pragma unroll
            for (int q = 0; q < 8; q++) { db0 += d0[q]; db1 += d1[q]; }
        }
        turn = turn == 0 ? a.gw - 1 : turn - 1;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            d0[q] *= sq[q]; d1[q] *= sq[q];
            if constexpr (FMT == GS4D_FMT_E4M3 || FMT == GS4D_FMT_E5M2) {
                const float4 f = lb_decode4<FMT>(cur.c[q]);
                c0[q] = f.x; c1[q] = f.y;
            } else if constexpr (FMT == GS4D_FMT_UINT8) { c0[q] = (float)(cur.c[q] & 255u); c1[q] = (float)(cur.c[q] >> 8); }
            else { c0[q] = (float)(int)(signed char)cur.c[q]; c1[q] = (float)((int)(short)cur.c[q] >> 8); }
        }
        uint4 da[2][TERMS], cc[2][1];
        split8<1, false>(c0, cc[0]);
        split8<1, false>(c1, cc[1]);
        if constexpr (ANY) {                              // infinities and NaNs: stand_in()
            auto split = [&](float (&d)[8], uint4 (&o)[TERMS]) {
                unsigned e[8];
#pragma unroll
                for (int q = 0; q < 8; q++) { e[q] = __float_as_uint(d[q]); d[q] = is_finite(e[q]) ? d[q] : stand_in(e[q]); }
                split8<TERMS, false>(d, o);
                const uint4 sp = specials8(e);            // (the codes are one term)
                o[TERMS - 1] = make_uint4(o[TERMS - 1].x | sp.x, o[TERMS - 1].y | sp.y, o[TERMS - 1].z | sp.z, o[TERMS - 1].w | sp.w);
            };
            split(d0, da[0]);
            split(d1, da[1]);
        } else {
            split8<TERMS, false>(d0, da[0]);
            split8<TERMS, false>(d1, da[1]);
        }
#pragma unroll
        for (int u = TERMS - 1; u >= 0; u--)
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int y = 0; y < 2; y++) acc[t][y] = mfma<LbBf16>(da[t][u], cc[y][0], acc[t][y]);
    };
    auto sweep = [&](auto any) {
        // whole steps of 16 rows, the next one in flight; the chunk's last, shorter step follows
        const long long stride = 16ll * slices, end = n1 - 15;
        long long r0 = n0 + 16 * slice;
        if (r0 < end) {
            // three steps in flight: with one, a step took as long as its loads (1.2 M x 256 -> 64 358 us, with three 280 at that time)
            Rows ring[3];
            load(ring[0], r0, Int<0>());
            load(ring[1], r0 + stride < end ? r0 + stride : r0, Int<0>());
            for (bool more = true; more;) {
#pragma unroll
                for (int u = 0; u < 3; u++) {
                    load(ring[(u + 2) % 3], r0 + 2 * stride < end ? r0 + 2 * stride : r0, Int<0>());
                    add(ring[u], r0, Int<0>(), any);
                    r0 += stride;
                    if (r0 >= end) { more = false; break; }
                }
            }
        }
        if (r0 < n1) {
            Rows cur;
            load(cur, r0, Int<1>());
            add(cur, r0, Int<1>(), any);
        }
    };
    if (mine) {
        sweep(Int<0>());
        // an infinity has left NaNs (its remainder is one): the wave's rows once more, with what that costs
        bool nan = false;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int y = 0; y < 2; y++)
#pragma unroll
                for (int r = 0; r < 16; r++) nan |= acc[t][y][r] != acc[t][y][r];
        if (__builtin_amdgcn_ballot_w64(nan)) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int y = 0; y < 2; y++) acc[t][y] = f32x16{};
            db0 = db1 = 0.f;
            turn = wave % a.gw;
            sweep(Int<1>());
        }
    }
    // ---- the slices of a group, in a fixed order: the upper half adds to the lower half until one is left
    for (int n = slices; n > 1; n >>= 1) {
        const int half = n >> 1;
        __syncthreads();
        if (slice >= half && slice < n) {
            float* p = s_red[(slice - half) * a.gw + wave % a.gw];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int r = 0; r < 16; r++) p[((t * 2 + y) * 16 + r) * 64 + lane] = acc[t][y][r];
        }
        __syncthreads();
        if (slice < half) {
            const float* p = s_red[slice * a.gw + wave % a.gw];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[t][y][r] += p[((t * 2 + y) * 16 + r) * 64 + lane];
        }
    }
    const size_t cell = (size_t)chunk * a.mtiles + mt;
    if (slice == 0 && mine) {
        float* p = a.slabs + (cell * a.groups + g) * 4096;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int y = 0; y < 2; y++)
#pragma unroll
                for (int r = 0; r < 16; r++) p[((t * 2 + y) * 16 + r) * 64 + lane] = acc[t][y][r];
    }
    if (z == 0) {                                         // db: each of the 8 waves has the column sums of its turns
        db0 += __shfl_xor(db0, 32, 64);
        db1 += __shfl_xor(db1, 32, 64);
        if (h == 0) { s_db[wave][2 * i] = db0; s_db[wave][2 * i + 1] = db1; }
        __syncthreads();
        if (tid < 64) {
            float s = 0.f;
            for (int q = 0; q < 8; q++) s += s_db[q][tid];
            a.slabs[(size_t)a.chunks * a.mtiles * a.groups * 4096 + cell * 64 + tid] = s;
        }
    }
}

// db alone (a frozen weight): the same sums in the same order as linear8_dw_kernel's, so that freezing changes no bit of them
template <typename T>
__global__ __launch_bounds__(512) void linear8_db_kernel(DwArgs a)
{
    __shared__ float s_db[8][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 31, h = lane >> 5;
    const int chunk = blockIdx.x % a.chunks, mt = blockIdx.x / a.chunks;
    const long long n0 = chunk * a.per, n1 = n0 + a.per < a.N ? n0 + a.per : a.N;
    const int m0 = min(mt * 64 + 2 * i, a.M - 1), m1 = min(mt * 64 + 2 * i + 1, a.M - 1);
    const T* __restrict__ dy = (const T*)a.dy;
    float d0 = 0.f, d1 = 0.f;
    // wave slice * gw + turn of 8: the steps of its slice, every gw-th from `turn` on
    const int slices = 8 / a.gw, slice = wave / a.gw, turn = wave % a.gw;
    for (long long r0 = n0 + 16 * (slice + (long long)slices * turn); r0 < n1; r0 += 128) {
        float v0[8], v1[8];
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const long long n = r0 + 8 * h + q, row = n < a.N ? n : a.N - 1;
            v0[q] = lb_load(dy[row * a.M + m0]);
            v1[q] = lb_load(dy[row * a.M + m1]);
        }
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const bool in = r0 + 8 * h + q < n1;
            d0 += in ? v0[q] : 0.f;
            d1 += in ? v1[q] : 0.f;
        }
    }
    d0 += __shfl_xor(d0, 32, 64);
    d1 += __shfl_xor(d1, 32, 64);
    if (h == 0) { s_db[wave][2 * i] = d0; s_db[wave][2 * i + 1] = d1; }
    __syncthreads();
    if (threadIdx.x < 64) {
        float s = 0.f;
        for (int q = 0; q < 8; q++) s += s_db[q][threadIdx.x];
        a.slabs[((size_t)chunk * a.mtiles + mt) * 64 + threadIdx.x] = s;
    }
}

// The slabs' sum, chunks in a fixed order (8 runs of them side by side), to the caller's arrays.
template <typename T>
__global__ __launch_bounds__(256) void linear8_dw_sum_kernel(DwArgs a, T* __restrict__ dw, T* __restrict__ db)
{
    __shared__ float part[8][32];
    const int o = threadIdx.x & 31, q = threadIdx.x >> 5;
    const long long cells = (long long)a.mtiles * a.groups * 4096, total = cells + a.mtiles * 64, e = (long long)blockIdx.x * 32 + o;
    const bool bias = e >= cells;
    const float* __restrict__ p = bias ? a.slabs + a.chunks * cells + (min(e, total - 1) - cells) : a.slabs + e;
    const long long step = bias ? a.mtiles * 64 : cells;
    const int per = (a.chunks + 7) / 8, c0 = q * per, c1 = min(a.chunks, c0 + per);
    float s = 0.f;
    for (int c = c0; c < c1; c += 8) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = p[min(c + u, c1 - 1) * step];
#pragma unroll
        for (int u = 0; u < 8; u++) s += c + u < c1 ? v[u] : 0.f;
    }
    part[q][o] = s;
    __syncthreads();
    if (q != 0 || e >= total) return;
    s = 0.f;
#pragma unroll
    for (int u = 0; u < 8; u++) s += part[u][o];
    if (bias) {
        const int m = (int)(e - cells);
        if (db && m < a.M) db[m] = lb_store<T>(s);
    } else if (dw) {
        const int lane = (int)(e & 63), r = (int)(e >> 6) & 15, y = (int)(e >> 10) & 1, t = (int)(e >> 11) & 1;
        const int g = (int)((e >> 12) % a.groups), mt = (int)((e >> 12) / a.groups);
        const int m = mt * 64 + 2 * ((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) + t, k = g * 64 + 2 * (lane & 31) + y;
        if (m < a.M && k < a.K) dw[(size_t)m * a.K + k] = lb_store<T>(s);
    }
}

#define LB_CUS 256

// how the weight gradient is cut: about one workgroup per CU, but at least 128 rows per chunk
static DwArgs dw_plan(long long N, int K, int M)
{
    DwArgs a = {};
    a.N = N; a.K = K; a.M = M;
    a.mtiles = (M + 63) / 64;
    a.groups = (K + 63) / 64;
    a.gw = a.groups >= 8 ? 8 : a.groups >= 4 ? 4 : a.groups >= 2 ? 2 : 1;
    const long long blocks = (long long)a.mtiles * ((a.groups + a.gw - 1) / a.gw);
    long long chunks = blocks >= LB_CUS ? 1 : LB_CUS / blocks;
    if (chunks > (N + 127) / 128) chunks = (N + 127) / 128;
    if (chunks < 1) chunks = 1;
    a.per = ((N + chunks - 1) / chunks + 127) / 128 * 128;
    if (a.per < 128) a.per = 128;
    a.chunks = (int)((N + a.per - 1) / a.per);
    if (a.chunks < 1) a.chunks = 1;
    return a;
}

static int check_cache(const gs4d_rows8* c, const char* who)
{
    if (!c || !c->codes || !c->scales || c->capacity < 1 || c->width < 1 || c->width > 65536 || c->pitch < c->width || (c->pitch & 15) ||
        ((uintptr_t)c->codes & 15) || ((uintptr_t)c->scales & 3) ||
        (c->group != 32 && c->group != 64 && c->group != 128) || c->fmt < GS4D_FMT_INT8 || c->fmt > GS4D_FMT_E5M2) {
        gs4d_set_error("%s: bad cache (1 to 65536 columns, pitch and codes multiples of 16 bytes, group 32, 64 or 128)", who);
        return GS4D_EINVAL;
    }
    return GS4D_OK;
}

static int check_rows(const gs4d_rows8* c, const void* rows, int dtype, long long ld, long long n, const void* slots, int slot_bytes,
                      long long start, const char* who)
{
    if (check_cache(c, who)) return GS4D_EINVAL;
    if (n < 0 || n > 2147483646ll || dtype < GS4D_F32 || dtype > GS4D_F16 || (n > 0 && (!rows || ld < c->width)) ||
        (slots ? slot_bytes != 4 && slot_bytes != 8 : start < 0 || start > c->capacity || n > c->capacity - start)) {
        gs4d_set_error("%s: bad rows or slots (rows in order must lie inside the cache)", who);
        return GS4D_EINVAL;
    }
    return GS4D_OK;
}

// a launch holds 2^32 work items; wide rows take a workgroup each
static bool too_many_rows(const gs4d_rows8* c, long long n, const char* who)
{
    if (c->width < 2048 || n < 1ll << 24) return false;
    gs4d_set_error("%s: %lld rows of %d columns are too many for one call", who, n, c->width);
    return true;
}

// items per row -> rows per workgroup, workgroups and the multiplier of the division by cpr
struct RowItems { int cpr, rpb; unsigned rcp, grid; };
static RowItems row_items(int cpr, long long n)
{
    RowItems r;
    r.cpr = cpr;
    r.rpb = cpr >= ROWS8_ITEMS ? 1 : ROWS8_ITEMS / cpr < ROWS8_ROWS ? ROWS8_ITEMS / cpr : ROWS8_ROWS;
    while (r.rpb > 1 && (n + r.rpb - 1) / r.rpb < 512) r.rpb = (r.rpb + 1) / 2;      // few rows: two workgroups per CU before long ones
    r.rcp = cpr > 1 ? (unsigned)((0x100000000ull + cpr - 1) / cpr) : 0;
    r.grid = (unsigned)((n + r.rpb - 1) / r.rpb);
    return r;
}

}  // namespace

extern "C" {

int gs4d_rows8_write(const gs4d_rows8* c, const void* rows, int dtype, long long ld, long long n, const void* slots, int slot_bytes,
                     long long start, void* stream)
{
    GS4D_TRACE_SCOPE("gs4d_rows8_write");
    hipStream_t s = (hipStream_t)stream;
    if (check_rows(c, rows, dtype, ld, n, slots, slot_bytes, start, "gs4d_rows8_write")) return GS4D_EINVAL;
    if (n == 0) return GS4D_OK;
    if (too_many_rows(c, n, "gs4d_rows8_write")) return GS4D_EINVAL;
    // rows for one slot: up to 256 rows each workgroup looks by itself (256 rows of 64: 3.2 us, with the owner array 5.2)
    const int dup = !slots || n == 1 ? 0 : n <= GS4D_ROWS8_SCAN ? 1 : 2;
    if (dup == 2 && !c->owner) { gs4d_set_error("gs4d_rows8_write: %lld rows at given slots need the cache's owner array", n); return GS4D_EINVAL; }
    const unsigned ogrid = (unsigned)((n + 255) / 256);
    auto with_slots = [&](auto tag) {
        using S = decltype(tag);
        const S* sl = (const S*)slots;
        if (dup == 2) hipLaunchKernelGGL(rows8_owner_kernel<S>, dim3(ogrid), dim3(256), 0, s, *c, sl, n);
        by_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int COLS = 16 / (int)sizeof(T);
            // lanes per group; a row shorter than a group takes as few as hold it
            const int groups = lb_groups(c->width, c->group);
            int lshift = 0;
            while ((COLS << lshift) < (groups > 1 ? c->group : c->width)) lshift++;
            const RowItems it = row_items(groups << lshift, n);
            return by_fmt(c->fmt, [&](auto f) {
                constexpr int F = decltype(f)::value;
                auto go = [&](auto full) {
                    constexpr bool FULL = decltype(full)::value != 0;
                    hipLaunchKernelGGL((rows8_write_kernel<F, T, S, FULL>), dim3(it.grid), dim3(256), 0, s, *c, (const T*)rows, ld, n, sl, start, it.cpr, it.rpb, it.rcp, lshift, dup);
                };
                if (c->width % COLS == 0) go(Int<1>());
                else go(Int<0>());
                return 0;
            });
        });
    };
    if (slots && slot_bytes == 4) with_slots(int());
    else with_slots((long long)0);
    GS4D_LAUNCH_CHECK("rows8_write", 0, s);
    return GS4D_OK;
}

int gs4d_rows8_read(const gs4d_rows8* c, void* out, int dtype, long long ld, long long n, const void* slots, int slot_bytes,
                    long long start, void* stream)
{
    GS4D_TRACE_SCOPE("gs4d_rows8_read");
    hipStream_t s = (hipStream_t)stream;
    if (check_rows(c, out, dtype, ld, n, slots, slot_bytes, start, "gs4d_rows8_read")) return GS4D_EINVAL;
    if (n == 0) return GS4D_OK;
    if (too_many_rows(c, n, "gs4d_rows8_read")) return GS4D_EINVAL;
    const int gshift = c->group == 32 ? 5 : c->group == 64 ? 6 : 7;
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int COLS = 16 / (int)sizeof(T);
        const RowItems it = row_items((c->width + COLS - 1) / COLS, n);
        return by_fmt(c->fmt, [&](auto f) {
            constexpr int F = decltype(f)::value;
            auto go = [&](auto tag, auto full) {
                using S = decltype(tag);
                hipLaunchKernelGGL((rows8_read_kernel<F, T, S, decltype(full)::value != 0>), dim3(it.grid), dim3(256), 0, s, *c, (T*)out, ld, n, (const S*)slots, start, it.cpr, it.rpb, it.rcp, gshift);
            };
            const bool narrow = slots && slot_bytes == 4;
            if (c->width % COLS == 0) { if (narrow) go(int(), Int<1>()); else go((long long)0, Int<1>()); }
            else { if (narrow) go(int(), Int<0>()); else go((long long)0, Int<0>()); }
            return 0;
        });
    });
    GS4D_LAUNCH_CHECK("rows8_read", 0, s);
    return GS4D_OK;
}

static int check_linear(int dtype, long long N, int K, int M, int fmt, const char* who)
{
    if (dtype < GS4D_F32 || dtype > GS4D_F16 || N < 0 || N > 2147483647ll || K < 1 || M < 1 || K > 1 << 20 || M > 1 << 20 ||
        (long long)K * M > 1ll << 28 ||
        fmt < GS4D_FMT_INT8 || fmt > GS4D_FMT_E5M2) {
        gs4d_set_error("%s: unsupported sizes or types", who);
        return GS4D_EINVAL;
    }
    return GS4D_OK;
}

size_t gs4d_linear8_keep_bytes(long long N, int K, int what)
{
    size_t bytes = 0;
    if (N < 0 || K < 1) return 0;
    carve_keep(nullptr, N, K, what, &bytes);
    return bytes;
}

size_t gs4d_linear8_scratch_bytes(long long N, int K, int M)
{
    if (N < 0 || K < 1 || M < 1) return 0;
    const DwArgs a = dw_plan(N, K, M);
    return (size_t)a.chunks * a.mtiles * ((size_t)a.groups * 4096 + 64) * sizeof(float) + 256;
}

}  // extern "C"

namespace {

// the products over the rows: NT tiles of 32 features per wave and as many groups of the weight in LDS as fit
template <typename T, bool DX>
static int launch_rows(RowsArgs& a, hipStream_t s)
{
    constexpr int LDS = 144 * 1024;
    const bool vec = a.C % 8 == 0;
    // tiles per wave: as wide as the registers allow, so that the rows are read and split seldom (65536 x 512 -> 512 fp16: 4 tiles
    // 71 us, 2 tiles 98), and no empty ones
    const int nt = sizeof(T) == 4 ? (a.F <= 32 ? 1 : 2) : a.F <= 64 ? 2 : 4;
    a.groups = (a.C + 63) / 64;
    const int per = 4 * nt * kTerms<T> * 1024;
    a.chunk = LDS / per < a.groups ? LDS / per : a.groups;
    // a contraction of one group: a workgroup takes as many of the column blocks as its LDS holds (a row's result in one go)
    const int all = (a.F + nt * 32 - 1) / (nt * 32);
    const long long ntile = (a.N + 31) / 32;
    const size_t joined = (size_t)(a.groups < 8 ? a.groups : 8) * (nt < 2 ? nt : 2) * 4096;
    // up to two rounds of tiles (float32; one and a bit for the 16-bit types, whose groups are shorter work), measured against ROWS_MANY:
    // float32 8192 x 256 -> 64 15 us against 23, 16384 19 against 23, 32768 26 against 25; bf16 8192 x 384 -> 128 12 against 16, 16384 the same
    const bool split = a.groups > 1 && ntile * 4 <= (sizeof(T) == 4 ? 8 : 5) * (LB_CUS / all) && (size_t)a.groups * per + joined <= 160 * 1024;
    const int mode = split ? ROWS_SPLIT : a.groups > 1 ? ROWS_MANY : all > 1 ? ROWS_WIDE : ROWS_ONE;
    a.blocks = mode == ROWS_WIDE ? (LDS / per < all ? LDS / per : all) : 1;
    a.ncb = (all + a.blocks - 1) / a.blocks;
    if (split) a.chunk = a.groups;
    const size_t lds = (size_t)a.chunk * a.blocks * per + (split ? joined : 0);
    auto launch = [&](auto n, auto v, auto o) {
        constexpr int THREADS = kRowsThreads<T, decltype(n)::value, decltype(v)::value != 0, decltype(o)::value>;
        auto k = linear8_rows_kernel<T, decltype(n)::value, decltype(v)::value != 0, DX, decltype(o)::value>;
        // 16 waves per CU if registers and LDS allow, never more workgroups than row tiles
        long long nwg = LB_CUS * (THREADS == 512 && lds <= 78 * 1024 ? 2 : 1) / a.ncb;
        if (nwg > ntile) nwg = ntile;
        if (nwg < 1) nwg = 1;
        if (nwg >= 8) nwg = nwg / 8 * 8;
        a.nwg = (int)nwg;
        if (lds > 64 * 1024) GS4D_HIP_CHECK(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(k, dim3((unsigned)(a.nwg * a.ncb)), dim3(THREADS), lds, s, a);
        return GS4D_OK;
    };
    auto with_nt = [&](auto n) {
        auto with_mode = [&](auto v) { return mode == ROWS_SPLIT ? launch(n, v, Int<ROWS_SPLIT>()) : mode == ROWS_MANY ? launch(n, v, Int<ROWS_MANY>()) : mode == ROWS_WIDE ? launch(n, v, Int<ROWS_WIDE>()) : launch(n, v, Int<ROWS_ONE>()); };
        return vec ? with_mode(Int<1>()) : with_mode(Int<0>());
    };
    if (nt == 2) return with_nt(Int<2>());
    if constexpr (sizeof(T) == 2) return with_nt(Int<4>());
    else return with_nt(Int<1>());
}

template <typename T>
static int launch_dw(DwArgs& a, int fmt, void* dw, void* db, hipStream_t s)
{
    if (dw) {
        const bool vec = a.M > 1;
        const unsigned grid = (unsigned)(a.chunks * a.mtiles * ((a.groups + a.gw - 1) / a.gw));
        by_fmt(fmt, [&](auto f) {
            constexpr int F = decltype(f)::value;
            auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3(grid), dim3(512), 0, s, a); };
            if (vec) go(linear8_dw_kernel<T, F, true>); else go(linear8_dw_kernel<T, F, false>);
            return 0;
        });
    } else {
        hipLaunchKernelGGL(linear8_db_kernel<T>, dim3((unsigned)(a.chunks * a.mtiles)), dim3(512), 0, s, a);
        a.groups = 0;                                     // the slabs hold db alone
    }
    const long long total = (long long)a.mtiles * a.groups * 4096 + a.mtiles * 64;
    hipLaunchKernelGGL(linear8_dw_sum_kernel<T>, dim3((unsigned)((total + 31) / 32)), dim3(256), 0, s, a, (T*)dw, (T*)db);
    return GS4D_OK;
}

}  // namespace

extern "C" {

int gs4d_linear8_forward(int dtype, long long N, int K, int M, const void* x, long long ldx, const void* w, const void* b, int relu,
                         int fmt, void* y, char* keep, int what, void* stream)
{
    GS4D_TRACE_SCOPE("gs4d_linear8_forward");
    hipStream_t s = (hipStream_t)stream;
    if (check_linear(dtype, N, K, M, fmt, "gs4d_linear8_forward")) return GS4D_EINVAL;
    if (N == 0) return GS4D_OK;
    if (!x || !w || !y || ldx < K || (what && (!keep || ((uintptr_t)keep & 255))) || ((what & GS4D_KEEP_SIGNS) && !relu)) {
        gs4d_set_error("gs4d_linear8_forward: null or misaligned pointer, or a row pitch below K");
        return GS4D_EINVAL;
    }
    RowsArgs a = {};
    a.N = N; a.C = K; a.F = M;
    a.x = x; a.ldx = ldx; a.w = w; a.wf = K; a.wc = 1; a.bias = b; a.y = y;
    a.lowest = relu ? 0 : (int)0x80000000;
    if (what) a.keep = carve_keep(keep, N, K, what, nullptr);
    a.fmt = relu && fmt == GS4D_FMT_INT8 ? GS4D_FMT_UINT8 : fmt;
    const int rc = by_type(dtype, [&](auto t) {
        if (few(dtype, false, N, K, M)) {
            const unsigned keepers = what ? (unsigned)((FEW_ROWS * (a.keep.kp / 64) + 15) / 16) : 0;
            hipLaunchKernelGGL(linear8_few_kernel<decltype(t)>, dim3((unsigned)((M + 15) / 16) + keepers, (unsigned)((N + FEW_ROWS - 1) / FEW_ROWS)), dim3(256), 0, s, a);
            return GS4D_OK;
        }
        return launch_rows<decltype(t), false>(a, s);
    });
    if (rc) return rc;
    GS4D_LAUNCH_CHECK("linear8_forward", 0, s);
    return GS4D_OK;
}

int gs4d_linear8_backward(int dtype, long long N, int K, int M, const void* dy, const void* w, int relu, int fmt, char* keep, int what,
                          void* dx, void* dw, void* db, char* scratch, void* stream)
{
    GS4D_TRACE_SCOPE("gs4d_linear8_backward");
    hipStream_t s = (hipStream_t)stream;
    if (check_linear(dtype, N, K, M, fmt, "gs4d_linear8_backward")) return GS4D_EINVAL;
    if ((N > 0 && !dy) || (dx && (!w || (relu && !(what & GS4D_KEEP_SIGNS)))) || (dw && !(what & GS4D_KEEP_CODES)) ||
        (what && N > 0 && (!keep || ((uintptr_t)keep & 255))) || ((dw || db) && (!scratch || ((uintptr_t)scratch & 255)))) {
        gs4d_set_error("gs4d_linear8_backward: null or misaligned pointer, or what the gradient needs was not kept");
        return GS4D_EINVAL;
    }
    const Keep kp = what && keep ? carve_keep(keep, N, K, what, nullptr) : Keep{};
    int rc = GS4D_OK;
    if (dx && N > 0) {
        RowsArgs a = {};
        a.N = N; a.C = M; a.F = K;
        a.x = dy; a.ldx = M; a.w = w; a.wf = 1; a.wc = K; a.y = dx;
        a.lowest = (int)0x80000000;
        if (relu) a.keep = kp;
        rc = by_type(dtype, [&](auto t) {
            if (few(dtype, true, N, K, M)) {
                hipLaunchKernelGGL(linear8_few_dx_kernel<decltype(t)>, dim3((unsigned)((K + 63) / 64), (unsigned)((N + FEW_ROWS - 1) / FEW_ROWS)), dim3(256), 0, s, a);
                return GS4D_OK;
            }
            return launch_rows<decltype(t), true>(a, s);
        });
        if (rc) return rc;
    }
    if (dw || db) {
        DwArgs a = dw_plan(N, K, M);
        a.dy = dy; a.keep = kp; a.slabs = (float*)scratch;
        rc = by_type(dtype, [&](auto t) { return launch_dw<decltype(t)>(a, relu && fmt == GS4D_FMT_INT8 ? GS4D_FMT_UINT8 : fmt, dw, db, s); });
        if (rc) return rc;
    }
    GS4D_LAUNCH_CHECK("linear8_backward", 0, s);
    return GS4D_OK;
}

}  // extern "C"

int gs4d_launch_keep(const Gs4dKeepJobs& jobs, long long rows, bool write, hipStream_t s)
{
    const dim3 grid((unsigned)((rows + 63) / 64), (unsigned)jobs.group0[jobs.n]);
    if (write) hipLaunchKernelGGL(keep_jobs_kernel<true>, grid, dim3(256), 0, s, jobs, rows);
    else hipLaunchKernelGGL(keep_jobs_kernel<false>, grid, dim3(256), 0, s, jobs, rows);
    GS4D_LAUNCH_CHECK("keep_jobs", 0, s);
    return GS4D_OK;
}
