// Rows in 8 bits (definition: lowbit.h): a cache of rows that are quantised as they are written, and a linear layer that keeps
// its input in 8 bits for its backward.
#include "lowbit.h"

namespace {

// ------------------------------------------------------------------ row cache
// A thread owns 8 consecutive columns, so a group is 4, 8 or 16 neighbouring lanes and its maximum a few lane exchanges.  A
// workgroup owns rpb rows; a row of more than 256 chunks is walked in steps of 256.
template <int FMT, int LANES, typename T, typename S>
__global__ __launch_bounds__(256) void rows8_write_kernel(gs4d_rows8 c, const T* __restrict__ rows, long long ld, long long n,
                                                          const S* __restrict__ slots, long long start, int cpr, int rpb, int dup)
{
    const int r = cpr >= 256 ? 0 : (int)threadIdx.x / cpr, ch0 = cpr >= 256 ? (int)threadIdx.x : (int)threadIdx.x % cpr;
    const long long i = (long long)blockIdx.x * rpb + r;
    if (r >= rpb || i >= n) return;
    const long long slot = slots ? (long long)slots[i] : start + i;
    if (slot < 0 || slot >= c.capacity) return;
    if (dup == 1) {                                      // few rows: is this the last one of its slot?
        for (long long j = i + 1; j < n; j++)
            if ((long long)slots[j] == slot) return;
    } else if (dup == 2) {
        if (c.owner[slot] != (int)(i + 1)) return;
    }
    const T* __restrict__ x = rows + i * ld;
    const int ng = (c.width + c.group - 1) / c.group;
    for (int ch = ch0; ch < cpr; ch += 256) {
        const int col = ch * 8;
        float v[8];
        unsigned m = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            v[q] = col + q < c.width ? lb_load(x[col + q]) : 0.f;
            m = max(m, lb_abs_bits(v[q]));
        }
#pragma unroll
        for (int s = 1; s < LANES; s <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, s, 64));
        const LbScale sc = lb_scale<FMT>(m);
        if (col < c.width) {
            uint2 w;
            w.x = lb_encode4<FMT>(v[0] * sc.inv, v[1] * sc.inv, v[2] * sc.inv, v[3] * sc.inv);
            w.y = lb_encode4<FMT>(v[4] * sc.inv, v[5] * sc.inv, v[6] * sc.inv, v[7] * sc.inv);
            *reinterpret_cast<uint2*>(c.codes + (size_t)slot * c.pitch + col) = w;
            if ((ch & (LANES - 1)) == 0) c.scales[(size_t)slot * ng + ch / LANES] = sc.s;
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

template <typename S>
__global__ __launch_bounds__(256) void rows8_owner_clear_kernel(gs4d_rows8 c, const S* __restrict__ slots, long long n)
{
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long slot = slots[i];
    if (slot >= 0 && slot < c.capacity) c.owner[slot] = 0;
}

template <int FMT, typename T, typename S>
__global__ __launch_bounds__(256) void rows8_read_kernel(gs4d_rows8 c, T* __restrict__ out, long long ld, long long n,
                                                         const S* __restrict__ slots, long long start, int cpr, int rpb)
{
    const int r = cpr >= 256 ? 0 : (int)threadIdx.x / cpr, ch0 = cpr >= 256 ? (int)threadIdx.x : (int)threadIdx.x % cpr;
    const long long i = (long long)blockIdx.x * rpb + r;
    if (r >= rpb || i >= n) return;
    const long long slot = slots ? (long long)slots[i] : start + i;
    const bool inside = slot >= 0 && slot < c.capacity;
    const int ng = (c.width + c.group - 1) / c.group;
    for (int ch = ch0; ch < cpr; ch += 256) {
        const int col = ch * 8;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        float s = 0.f;
        if (inside) {
            const uint2 w = *reinterpret_cast<const uint2*>(c.codes + (size_t)slot * c.pitch + col);
            s = c.scales[(size_t)slot * ng + col / c.group];
            a = lb_decode4<FMT>(w.x);
            b = lb_decode4<FMT>(w.y);
        }
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int q = 0; q < 8; q++)
            if (col + q < c.width) out[i * ld + col + q] = lb_store<T>(s * v[q]);
    }
}

// ------------------------------------------------------------------ linear
// What the backward keeps of the input, in one block: codes [N][kp] | scales [N][kp / 64] | sign bits [N][kp / 8] (bit k & 7 of
// byte k >> 3: x > 0), kp = K rounded up to 64.
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

// relu that keeps a NaN
__device__ __forceinline__ float lb_relu(float x) { return x < 0.f ? 0.f : x; }

template <int FMT, bool RELU, typename T>
__global__ __launch_bounds__(256) void linear8_keep_kernel(Keep kp, const T* __restrict__ x, long long ldx, long long N, int K)
{
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;       // 8 lanes per group of 64
    const int cpr = kp.kp / 8;
    const long long i = t / cpr;
    const int col = (int)(t % cpr) * 8;
    if (i >= N) return;
    float v[8];
    unsigned m = 0, bits = 0;
#pragma unroll
    for (int q = 0; q < 8; q++) {
        v[q] = col + q < K ? lb_load(x[i * ldx + col + q]) : 0.f;
        if (RELU) {
            bits |= (v[q] <= 0.f ? 0u : 1u) << q;
            v[q] = lb_relu(v[q]);
        }
        m = max(m, lb_abs_bits(v[q]));
    }
    if (RELU && kp.bits) kp.bits[i * cpr + (col >> 3)] = (unsigned char)bits;
    if (!kp.codes) return;
#pragma unroll
    for (int s = 1; s < 8; s <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, s, 64));
    const LbScale sc = lb_scale<FMT>(m);
    uint2 w;
    w.x = lb_encode4<FMT>(v[0] * sc.inv, v[1] * sc.inv, v[2] * sc.inv, v[3] * sc.inv);
    w.y = lb_encode4<FMT>(v[4] * sc.inv, v[5] * sc.inv, v[6] * sc.inv, v[7] * sc.inv);
    *reinterpret_cast<uint2*>(kp.codes + (size_t)i * kp.kp + col) = w;
    if ((col & 63) == 0) kp.scales[(size_t)i * (kp.kp / 64) + (col >> 6)] = sc.s;
}

// The three products, simplest form: a 64 x 64 tile of the result per workgroup, 16 steps of the contraction at a time through
// LDS, 4 x 4 results per thread in float32.  LA(row, k) and LB(col, k) give the operands, out-of-range ones as zero.
template <typename LA, typename LB, typename ST>
__device__ __forceinline__ void tile_product(long long k0, long long k1, LA la, LB lb, ST st)
{
    __shared__ float sa[16][65], sb[16][65];
    const int tid = threadIdx.x, tr = (tid >> 4) * 4, tc = (tid & 15) * 4;
    float acc[4][4] = {};
    for (long long k = k0; k < k1; k += 16) {
        for (int e = tid; e < 1024; e += 256) {
            const int r = e >> 4, q = e & 15;
            sa[q][r] = la(r, k + q);
            sb[q][r] = lb(r, k + q);
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 16; q++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sa[q][tr + i], sb[q][tc + j], acc[i][j]);
        }
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) st(tr + i, tc + j, acc[i][j]);
}

template <bool RELU, typename T>
__global__ __launch_bounds__(256) void linear8_forward_kernel(long long N, int K, int M, const T* __restrict__ x, long long ldx,
                                                              const T* __restrict__ w, const T* __restrict__ b, T* __restrict__ y)
{
    const long long r0 = (long long)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64;
    tile_product(0, K,
        [&](int r, long long k) { const float v = r0 + r < N && k < K ? lb_load(x[(r0 + r) * ldx + k]) : 0.f; return RELU ? lb_relu(v) : v; },
        [&](int c, long long k) { return c0 + c < M && k < K ? lb_load(w[(long long)(c0 + c) * K + k]) : 0.f; },
        [&](int r, int c, float v) { if (r0 + r < N && c0 + c < M) y[(r0 + r) * M + c0 + c] = lb_store<T>(v + (b ? lb_load(b[c0 + c]) : 0.f)); });
}

template <typename T>
__global__ __launch_bounds__(256) void linear8_dx_kernel(long long N, int K, int M, const T* __restrict__ dy, const T* __restrict__ w,
                                                         Keep kp, T* __restrict__ dx)
{
    const long long r0 = (long long)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64;
    tile_product(0, M,
        [&](int r, long long m) { return r0 + r < N && m < M ? lb_load(dy[(r0 + r) * M + m]) : 0.f; },
        [&](int c, long long m) { return c0 + c < K && m < M ? lb_load(w[m * K + c0 + c]) : 0.f; },
        [&](int r, int c, float v) {
            if (r0 + r >= N || c0 + c >= K) return;
            const int k = c0 + c;
            if (kp.bits && !(kp.bits[(r0 + r) * (kp.kp / 8) + (k >> 3)] >> (k & 7) & 1)) v = 0.f;
            dx[(r0 + r) * K + k] = lb_store<T>(v);
        });
}

// partial[chunk][m][kc]: kc < K the weight gradient of the chunk's rows, kc == K the bias gradient
template <int FMT, typename T>
__global__ __launch_bounds__(256) void linear8_dw_kernel(long long N, int K, int M, const T* __restrict__ dy, Keep kp,
                                                         long long per, float* __restrict__ partial)
{
    const int m0 = blockIdx.y * 64, c0 = blockIdx.z * 64;
    const long long n0 = (long long)blockIdx.x * per, n1 = min(N, n0 + per);
    tile_product(n0, n1,
        [&](int r, long long n) { return m0 + r < M && n < n1 ? lb_load(dy[n * M + m0 + r]) : 0.f; },
        [&](int c, long long n) {
            const int k = c0 + c;
            if (n >= n1 || k > K) return 0.f;
            if (k == K) return 1.f;
            const unsigned wd = kp.codes[(size_t)n * kp.kp + k];
            return lb_decode4<FMT>(wd).x * kp.scales[(size_t)n * (kp.kp / 64) + (k >> 6)];
        },
        [&](int r, int c, float v) { if (m0 + r < M && c0 + c <= K) partial[((size_t)blockIdx.x * M + m0 + r) * (K + 1) + c0 + c] = v; });
}

template <typename T>
__global__ __launch_bounds__(256) void linear8_dw_sum_kernel(int K, int M, int chunks, const float* __restrict__ partial,
                                                             T* __restrict__ dw, T* __restrict__ db)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x, total = (long long)M * (K + 1);
    if (e >= total) return;
    float s = 0.f;
    for (int c = 0; c < chunks; c++) s += partial[(size_t)c * total + e];
    const int m = (int)(e / (K + 1)), k = (int)(e % (K + 1));
    if (k < K) { if (dw) dw[(size_t)m * K + k] = lb_store<T>(s); }
    else if (db) db[m] = lb_store<T>(s);
}

static long long dw_chunks(long long N) { return N <= 0 ? 1 : (N + 2047) / 2048 < 256 ? (N + 2047) / 2048 : 256; }

static int check_cache(const gs4d_rows8* c, const char* who)
{
    if (!c || !c->codes || !c->scales || c->capacity < 1 || c->width < 1 || c->pitch < c->width || (c->pitch & 15) ||
        ((uintptr_t)c->codes & 15) || ((uintptr_t)c->scales & 3) ||
        (c->group != 32 && c->group != 64 && c->group != 128) || c->fmt < GS4D_FMT_INT8 || c->fmt > GS4D_FMT_E5M2) {
        gs4d_set_error("%s: bad cache (pitch and codes must be multiples of 16 bytes, group 32, 64 or 128)", who);
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

}  // namespace

extern "C" {

int gs4d_rows8_write(const gs4d_rows8* c, const void* rows, int dtype, long long ld, long long n, const void* slots, int slot_bytes,
                     long long start, void* stream)
{
    GS4D_TRACE_SCOPE("gs4d_rows8_write");
    hipStream_t s = (hipStream_t)stream;
    if (check_rows(c, rows, dtype, ld, n, slots, slot_bytes, start, "gs4d_rows8_write")) return GS4D_EINVAL;
    if (n == 0) return GS4D_OK;
    const int dup = !slots || n == 1 ? 0 : n <= GS4D_ROWS8_SCAN ? 1 : 2;
    if (dup == 2 && !c->owner) { gs4d_set_error("gs4d_rows8_write: %lld rows at given slots need the cache's owner array", n); return GS4D_EINVAL; }
    const int cpr = lb_groups(c->width, c->group) * (c->group / 8), rpb = cpr >= 256 ? 1 : 256 / cpr;
    const unsigned grid = (unsigned)((n + rpb - 1) / rpb), ogrid = (unsigned)((n + 255) / 256);
    auto with_slots = [&](auto tag) {
        using S = decltype(tag);
        const S* sl = (const S*)slots;
        if (dup == 2) hipLaunchKernelGGL(rows8_owner_kernel<S>, dim3(ogrid), dim3(256), 0, s, *c, sl, n);
        by_type(dtype, [&](auto t) {
            using T = decltype(t);
            return by_fmt(c->fmt, [&](auto f) {
                constexpr int F = decltype(f)::value;
                auto k = c->group == 32 ? rows8_write_kernel<F, 4, T, S> : c->group == 64 ? rows8_write_kernel<F, 8, T, S> : rows8_write_kernel<F, 16, T, S>;
                hipLaunchKernelGGL(k, dim3(grid), dim3(256), 0, s, *c, (const T*)rows, ld, n, sl, start, cpr, rpb, dup);
                return 0;
            });
        });
        if (dup == 2) hipLaunchKernelGGL(rows8_owner_clear_kernel<S>, dim3(ogrid), dim3(256), 0, s, *c, sl, n);
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
    const int cpr = (c->width + 7) / 8, rpb = cpr >= 256 ? 1 : 256 / cpr;
    const unsigned grid = (unsigned)((n + rpb - 1) / rpb);
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        return by_fmt(c->fmt, [&](auto f) {
            constexpr int F = decltype(f)::value;
            if (slots && slot_bytes == 4)
                hipLaunchKernelGGL((rows8_read_kernel<F, T, int>), dim3(grid), dim3(256), 0, s, *c, (T*)out, ld, n, (const int*)slots, start, cpr, rpb);
            else
                hipLaunchKernelGGL((rows8_read_kernel<F, T, long long>), dim3(grid), dim3(256), 0, s, *c, (T*)out, ld, n, (const long long*)slots, start, cpr, rpb);
            return 0;
        });
    });
    GS4D_LAUNCH_CHECK("rows8_read", 0, s);
    return GS4D_OK;
}

static int check_linear(int dtype, long long N, int K, int M, int fmt, const char* who)
{
    if (dtype < GS4D_F32 || dtype > GS4D_F16 || N < 0 || N > 2147483647ll || K < 1 || M < 1 || K > 65535 * 64 || M > 65535 * 64 ||
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
    return (size_t)dw_chunks(N) * M * ((size_t)K + 1) * sizeof(float) + 256;
}

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
    const Keep kp = what ? carve_keep(keep, N, K, what, nullptr) : Keep{};
    const int kf = relu && fmt == GS4D_FMT_INT8 ? GS4D_FMT_UINT8 : fmt;
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (what)
            by_fmt(kf, [&](auto f) {
                constexpr int F = decltype(f)::value;
                const unsigned grid = (unsigned)(((size_t)N * (kp.kp / 8) + 255) / 256);
                auto k = relu ? linear8_keep_kernel<F, true, T> : linear8_keep_kernel<F, false, T>;
                hipLaunchKernelGGL(k, dim3(grid), dim3(256), 0, s, kp, (const T*)x, ldx, N, K);
                return 0;
            });
        auto k = relu ? linear8_forward_kernel<true, T> : linear8_forward_kernel<false, T>;
        hipLaunchKernelGGL(k, dim3((unsigned)((N + 63) / 64), (M + 63) / 64), dim3(256), 0, s, N, K, M, (const T*)x, ldx, (const T*)w, (const T*)b, (T*)y);
        return 0;
    });
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
    Keep masked = kp;
    if (!relu) masked.bits = nullptr;
    const int kf = relu && fmt == GS4D_FMT_INT8 ? GS4D_FMT_UINT8 : fmt;
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (dx && N > 0)
            hipLaunchKernelGGL(linear8_dx_kernel<T>, dim3((unsigned)((N + 63) / 64), (K + 63) / 64), dim3(256), 0, s, N, K, M, (const T*)dy, (const T*)w, masked, (T*)dx);
        if (dw || db) {
            const int chunks = (int)dw_chunks(N), Kw = dw ? K : 0;       // without dw: the bias column alone
            const long long per = (N + chunks - 1) / chunks;
            by_fmt(kf, [&](auto f) {
                constexpr int F = decltype(f)::value;
                hipLaunchKernelGGL((linear8_dw_kernel<F, T>), dim3(chunks, (M + 63) / 64, (Kw + 64) / 64), dim3(256), 0, s, N, Kw, M, (const T*)dy, kp, per, (float*)scratch);
                return 0;
            });
            hipLaunchKernelGGL(linear8_dw_sum_kernel<T>, dim3((unsigned)(((size_t)M * (Kw + 1) + 255) / 256)), dim3(256), 0, s, Kw, M, chunks, (const float*)scratch, (T*)dw, (T*)db);
        }
        return 0;
    });
    GS4D_LAUNCH_CHECK("linear8_backward", 0, s);
    return GS4D_OK;
}

}  // extern "C"
