// linear.cu — y = act(x W^T + b) + residual and its gradients: products on the multiply-add pipes, the sums
// over parts of a tile, the gradient of the activation, and the host's part.
//
//   z = x W^T + b;  y = act(z) + r;   v_z = v_y act'(z);  v_x = v_z W;  v_W = v_z^T x;  v_b = sum of v_z's rows.
// Three products of one kind, C = A B^T over an axis K along which either operand's rows or columns run.
#include <algorithm>

#include "sx_linear.h"

namespace sx {
namespace {

// ---- products on the multiply-add pipes ----
// A CTA takes TILE x TILE values of C (128, or 64 where there are few), a thread 8 x 8 of them as 2 x 2 blocks of
// 4 x 4; 16 of K at a time go through shared memory, the next 16 are on their way in registers meanwhile.
constexpr int kDepth = 16;
template <int TILE>
constexpr int kThreads = TILE * TILE / 64;

// The thread's share of a TILE x 16 block of an operand, 8 values at a time: along K for a row, or along the rows
// for a value of K.
template <int TILE>
struct Staged {
    static constexpr int kPitch = TILE + 4, kTurns = TILE * 2 / kThreads<TILE>;
    float x[kTurns][8];
    __device__ __forceinline__ void load(const LinearOperand& o, int64_t row0, int64_t rows, int64_t k0, int64_t k_end, bool wide) {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int t = threadIdx.x + i * kThreads<TILE>;
            const int64_t row = row0 + (o.across ? t % (TILE / 8) * 8 : t / 2), k = k0 + (o.across ? t / (TILE / 8) : t % 2 * 8);
            const float* p = static_cast<const float*>(o.data) + (o.across ? k * o.stride + row : row * o.stride + k);
            const int64_t left = (o.across ? k < k_end : row < rows) ? (o.across ? rows - row : k_end - k) : 0;
            if (wide && left >= 8) {
                *reinterpret_cast<float4*>(x[i]) = reinterpret_cast<const float4*>(p)[0];
                *reinterpret_cast<float4*>(x[i] + 4) = reinterpret_cast<const float4*>(p)[1];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][j] = j < left ? p[j] : 0.f;
            }
        }
    }
    __device__ __forceinline__ void store(const LinearOperand& o, float (&to)[kDepth][kPitch]) const {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int t = threadIdx.x + i * kThreads<TILE>;
            if (o.across) {
                float* at = &to[t / (TILE / 8)][t % (TILE / 8) * 8];
                *reinterpret_cast<float4*>(at) = *reinterpret_cast<const float4*>(x[i]);
                *reinterpret_cast<float4*>(at + 4) = *reinterpret_cast<const float4*>(x[i] + 4);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) to[t % 2 * 8 + j][t / 2] = x[i][j];
            }
        }
    }
};

// The epilogue for `n` (at most N) consecutive columns of a row.
template <typename T, int N>
__device__ __forceinline__ void linear_finish(const LinearProduct& p, int64_t row, int64_t col, float (&z)[N], const float (&bias)[N], int n) {
    T* to = static_cast<T*>(p.y) + row * p.y_stride + col;
    T* keep = static_cast<T*>(p.pre) + row * p.pre_stride + col;
    const T* add = static_cast<const T*>(p.residual) + row * p.residual_stride + col;
    const auto fits = [](const T* a) { return reinterpret_cast<uintptr_t>(a) % (N * sizeof(T)) == 0; };
    const bool whole = n == N && fits(to) && (!p.pre || fits(keep)) && (!p.residual || fits(add));
    Pack<T, N> r{};
    if (p.residual) {
        if (whole) {
            r = *reinterpret_cast<const Pack<T, N>*>(add);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) r.v[i] = add[i];
        }
    }
    Pack<T, N> pre, y;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        z[i] += bias[i];
        pre.v[i] = from_f32<T>(z[i]);
    }
    if (p.act != SXCUDA_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = act_of<T>(p.act, z[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) y.v[i] = from_f32<T>(p.residual ? z[i] + to_f32(r.v[i]) : z[i]);
    if (whole) {
        *reinterpret_cast<Pack<T, N>*>(to) = y;
        if (p.pre) *reinterpret_cast<Pack<T, N>*>(keep) = pre;
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i >= n) break;
        to[i] = y.v[i];
        if (p.pre) keep[i] = pre.v[i];
    }
}
template <int N>
__device__ __forceinline__ void linear_biases(const LinearProduct& p, int64_t col, int n, float (&bias)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) bias[i] = i < n ? linear_param(p.bias, p.bias_dtype, col + i) : 0.f;
}

// A launch's one product, or the backward's two, which have nothing to wait for in one another: small ones fill the
// SMs better together. Backward calls with two launches and with one, us: 604 x 77 x 913 33 and 28, 300 x 256 x 256 with
// relu 26 and 17, 2048 x 128 x 512 with gelu 37 and 35, 20000 x 64 x 64 36 and 29 (with one launch for the joins). A kernel
// that finds its product at run time is slower (forward 2048 x 128 x 512: 19 and 25), so one product has a kernel of its own.
template <int N>
struct LinearProducts {
    LinearProduct p[N];
    bool a_wide[N], b_wide[N];  // rows are read 16 bytes at a time
};

template <int TILE, int N>
__global__ void __launch_bounds__(kThreads<TILE>, TILE == 128 ? 2 : 6) linear_kernel(const __grid_constant__ LinearProducts<N> of) {
    const int32_t first = N == 2 ? of.p[0].plan.workers : 0, block = static_cast<int32_t>(blockIdx.x);
    const int which = N == 2 && block >= first;
    const LinearProduct& p = of.p[which];
    const bool a_wide = of.a_wide[which], b_wide = of.b_wide[which];
    constexpr int kSide = TILE / 8, kHalf = TILE / 2, kPitch = TILE + 4;
    __shared__ __align__(16) float smem[2][2][kDepth][kPitch];  // of A, of B; twice
    const int tx = threadIdx.x % kSide, ty = threadIdx.x / kSide;
    LinearWalk walk(p.plan, which ? block - first : block);
    LinearPiece piece;
    while (walk.next(p.plan, piece)) {
        const LinearTile tile = linear_tile(p.plan, piece.tile);
        const int64_t m0 = static_cast<int64_t>(tile.m) * TILE, n0 = static_cast<int64_t>(tile.n) * TILE, end = min(static_cast<int64_t>(piece.k1) * kDepth, p.k);
        tc::Two c[8][4];  // two columns each
#pragma unroll
        for (int i = 0; i < 32; ++i) c[i / 4][i % 4] = tc::two(0.f, 0.f);
        Staged<TILE> a, b;
        a.load(p.a, m0, p.m, static_cast<int64_t>(piece.k0) * kDepth, end, a_wide);
        b.load(p.b, n0, p.n, static_cast<int64_t>(piece.k0) * kDepth, end, b_wide);
        for (int k = piece.k0; k < piece.k1; ++k) {
            const int at = k & 1;
            a.store(p.a, smem[0][at]);
            b.store(p.b, smem[1][at]);
            __syncthreads();
            if (k + 1 < piece.k1) {
                a.load(p.a, m0, p.m, static_cast<int64_t>(k + 1) * kDepth, end, a_wide);
                b.load(p.b, n0, p.n, static_cast<int64_t>(k + 1) * kDepth, end, b_wide);
            }
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                float x[8];
                tc::Two y[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    *reinterpret_cast<float4*>(x + 4 * h) = *reinterpret_cast<const float4*>(&smem[0][at][d][ty * 4 + h * kHalf]);
                    const float4 v = *reinterpret_cast<const float4*>(&smem[1][at][d][tx * 4 + h * kHalf]);
                    y[2 * h] = tc::two(v.x, v.y), y[2 * h + 1] = tc::two(v.z, v.w);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[i][j] = tc::fma2(tc::two(x[i], x[i]), y[j], c[i][j]);
            }
        }
        // half of the rows at a time through shared memory: then 4 columns of row after row, with little code
        float(*rows)[kPitch] = reinterpret_cast<float(*)[kPitch]>(smem);
        const int col = static_cast<int>(threadIdx.x) % (TILE / 4) * 4, n = static_cast<int>(min(p.n - n0 - col, static_cast<int64_t>(4)));
        float bias[4];
        linear_biases(p, n0 + col, n, bias);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float4 v;
                    tc::split(c[4 * h + i][2 * j], v.x, v.y);
                    tc::split(c[4 * h + i][2 * j + 1], v.z, v.w);
                    *reinterpret_cast<float4*>(&rows[ty * 4 + i][tx * 4 + j * kHalf]) = v;
                }
            __syncthreads();
#pragma unroll 1
            for (int r = static_cast<int>(threadIdx.x) / (TILE / 4); r < kHalf; r += kThreads<TILE> / (TILE / 4)) {
                const int row = r + h * kHalf;
                if (m0 + row >= p.m || n <= 0) break;
                const float4 v = *reinterpret_cast<const float4*>(&rows[r][col]);
                float z[4] = {v.x, v.y, v.z, v.w};
                if (piece.slot < 0) linear_finish<float, 4>(p, m0 + row, n0 + col, z, bias, n);
                else *reinterpret_cast<float4*>(linear_part(p, piece.slot, row, col)) = v;
            }
        }
        __syncthreads();  // the next piece's first stores
    }
}

// Adds the parts of the tiles that are cut, in an order of K that the sizes alone decide, and finishes them. A unit
// is 8 rows by 32 columns, 256 bytes of a part side by side and 64 of a row of y, a lane's 8 columns of a row.
// blockIdx.y is the tile's number among those that are cut, blockIdx.z the product. With few parts of many tiles
// each warp adds a unit; where a tile has many, W = 8 or 32 warps share one, every W-th part each (backward calls with
// one warp a unit and with this, us: float32 20000 x 64 x 64, 313 parts, 57 and 31, 40000 x 3 x 64 105 and 47; bf16
// 40000 x 256 x 256 with gelu 65 and 55).
constexpr int join_warps(int w) { return w == 1 ? 8 : w; }
template <typename T, int N, int W>
__global__ void __launch_bounds__(32 * join_warps(W)) linear_join_kernel(const __grid_constant__ LinearProducts<N> of) {
    const LinearProduct& p = of.p[N == 2 ? blockIdx.z : 0];
    const LinearPlan& plan = p.plan;
    const int32_t t = static_cast<int32_t>(blockIdx.y);
    if (N == 2 && t >= plan.rest) return;
    const int32_t parts = plan.parts(t);
    const LinearTile tile = linear_tile(plan, plan.whole + t);
    const int64_t m0 = static_cast<int64_t>(tile.m) * plan.tile_m, n0 = static_cast<int64_t>(tile.n) * plan.tile_n;
    const int rows = static_cast<int>(min(static_cast<int64_t>(plan.tile_m), p.m - m0)), groups = plan.tile_n / 8;
    const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    const int at = W == 1 ? static_cast<int>(blockIdx.x) * 8 + warp : static_cast<int>(blockIdx.x);
    const int row = at / (groups / 4) * 8 + lane % 8, col = (at % (groups / 4) * 4 + lane / 8) * 8;
    const int64_t n = min(p.n - n0 - col, static_cast<int64_t>(8));
    const bool here = row < rows && n > 0;
    float z[8] = {};
    if (here) {
#pragma unroll 4
        for (int i = W == 1 ? 0 : warp; i < parts; i += W) {
            const float4* part = reinterpret_cast<const float4*>(linear_part(p, t * plan.slots + i, row, col));
            const float4 x = part[0], y = part[1];
            z[0] += x.x, z[1] += x.y, z[2] += x.z, z[3] += x.w;
            z[4] += y.x, z[5] += y.y, z[6] += y.z, z[7] += y.w;
        }
    }
    if constexpr (W > 1) {
        __shared__ float4 sums[W][2][32];
        sums[warp][0][lane] = make_float4(z[0], z[1], z[2], z[3]);
        sums[warp][1][lane] = make_float4(z[4], z[5], z[6], z[7]);
        __syncthreads();
        if (warp) return;
#pragma unroll 4
        for (int w = 1; w < W; ++w) {
            const float4 x = sums[w][0][lane], y = sums[w][1][lane];
            z[0] += x.x, z[1] += x.y, z[2] += x.z, z[3] += x.w;
            z[4] += y.x, z[5] += y.y, z[6] += y.z, z[7] += y.w;
        }
    }
    if (!here) return;
    float bias[8];
    linear_biases(p, n0 + col, static_cast<int>(n), bias);
    linear_finish<T, 8>(p, m0 + row, n0 + col, z, bias, static_cast<int>(n));
}

bool linear_wide(const LinearOperand& o, int64_t size) {
    return reinterpret_cast<uintptr_t>(o.data) % 16 == 0 && o.stride * size % 16 == 0;
}

}  // namespace

LinearPlan linear_plan(int64_t m, int64_t n, int64_t k, int tile_m, int tile_n, int depth, int64_t workers, int64_t least,
                       int64_t gain) {
    LinearPlan p;
    p.tile_m = tile_m, p.tile_n = tile_n;
    const int64_t tiles_m = (m + tile_m - 1) / tile_m, tiles_n = (n + tile_n - 1) / tile_n, tiles = tiles_m * tiles_n;
    if (tiles > INT32_MAX / kLinearBand) throw_invalid("linear", "too many tiles");
    const int64_t kblocks = (k + depth - 1) / depth, rest = tiles % workers;
    p.tiles_m = static_cast<int32_t>(tiles_m), p.tiles_n = static_cast<int32_t>(tiles_n);
    p.kblocks = static_cast<int32_t>(kblocks);
    p.workers = static_cast<int32_t>(std::min(tiles, workers));
    p.whole = static_cast<int32_t>(tiles);
    if (rest == 0) return p;
    const int64_t share = std::max(least, (rest * kblocks + workers - 1) / workers);
    if (kblocks - share < gain || rest * kblocks > INT32_MAX) return p;
    const int64_t main = std::min(workers / rest, kblocks / share), tail = kblocks - main * share, others = workers - main * rest;
    const int64_t tail_share = tail ? std::max(std::min(least, tail), (rest * tail + others - 1) / others) : 1;
    p.whole = static_cast<int32_t>(tiles - rest);
    p.rest = static_cast<int32_t>(rest);
    p.main = static_cast<int32_t>(main);
    p.share = static_cast<int32_t>(share);
    p.tail = static_cast<int32_t>(tail);
    p.tail_share = static_cast<int32_t>(tail_share);
    p.slots = static_cast<int32_t>(main + (tail ? (tail + tail_share - 1) / tail_share + 1 : 0));
    p.workers = static_cast<int32_t>(p.whole ? workers : main * rest + (rest * tail + tail_share - 1) / tail_share);
    return p;
}

namespace {

// float32: tiles of 128 do a large product in 0.9 of the time of tiles of 64, but need twice two turns of the SMs for
// that, and lose it where they reach 5% further beyond the sizes. 512 -> n features, 128 and 64 in us: 20000 rows,
// n = 96 113 and 89, 192 161 and 105, 384 222 and 202, 512 270 and 274, 700 381 and 363, 1024 487 and 539; 80000
// rows, 192 483 and 396, 256 486 and 541.
LinearPlan product_plan(int32_t dtype, int64_t m, int64_t n, int64_t k) {
    if (dtype != SXCUDA_F32) return linear_tc_plan(m, n, k);
    const auto tiles = [&](int64_t side) { return (m + side - 1) / side * ((n + side - 1) / side); };
    const int64_t sms = sm_count();
    const bool large = tiles(128) >= sms * 4 && tiles(128) * 4 * 20 <= tiles(64) * 21;
    return large ? linear_plan(m, n, k, 128, 128, kDepth, sms * 2, 8, 32) : linear_plan(m, n, k, 64, 64, kDepth, sms * 6, 4, 12);
}

int64_t join_units(const LinearProduct& p) { return (std::min<int64_t>(p.m, p.plan.tile_m) + 7) / 8 * (p.plan.tile_n / 32); }
int join_share(const LinearProduct& p) {
    if (p.plan.slots < 16) return 1;
    return p.plan.slots >= 64 && join_units(p) * p.plan.rest <= 128 ? 32 : 8;
}

template <int N>
LinearProducts<N> products_of(const LinearProduct (&p)[N]) {
    LinearProducts<N> of;
    for (int i = 0; i < N; ++i) of.p[i] = p[i], of.a_wide[i] = linear_wide(p[i].a, 4), of.b_wide[i] = linear_wide(p[i].b, 4);
    return of;
}
// Two products are joined by one launch where they are joined alike. Otherwise they have one each: for the sums not to
// depend on whether the other product is asked for, and as warps without a part cost more (3000 x 256 x 256 backward, one
// launch of warps with and without parts 52 us, two 41).
template <typename T, int N>
void launch_join(const LinearProducts<N>& of, cudaStream_t s) {
    if constexpr (N == 2) {
        if (!of.p[0].plan.cut() || !of.p[1].plan.cut() || join_share(of.p[0]) != join_share(of.p[1])) {
            for (const LinearProduct& p : of.p) launch_join<T>(products_of({p}), s);
            return;
        }
    }
    int64_t units = 0, rest = 0;
    for (const LinearProduct& p : of.p) units = std::max(units, join_units(p)), rest = std::max<int64_t>(rest, p.plan.rest);
    if (!rest) return;
    const auto run = [&](auto warps) {
        constexpr int W = decltype(warps)::value;
        const auto join = linear_join_kernel<T, N, W>;
        SX_LAUNCH(join, dim3(blocks_for(units, W == 1 ? 8 : 1), static_cast<unsigned>(rest), N), 32 * join_warps(W), 0, s, of);
    };
    const int share = join_share(of.p[0]);
    if (share == 32) run(std::integral_constant<int, 32>{});
    else if (share == 8) run(std::integral_constant<int, 8>{});
    else run(std::integral_constant<int, 1>{});
}

void launch_product(const LinearProduct& p, cudaStream_t s) {
    const LinearProducts<1> of = products_of({p});
    const auto run = [&](auto kernel, int threads) { SX_LAUNCH(kernel, static_cast<unsigned>(p.plan.workers), threads, 0, s, of); };
    if (p.dtype != SXCUDA_F32) launch_linear_tc(p, s);
    else if (p.plan.tile_m == 128) run(linear_kernel<128, 1>, kThreads<128>);
    else run(linear_kernel<64, 1>, kThreads<64>);
    by_dtype(p.dtype, [&](auto t) { launch_join<decltype(t)>(of, s); });
}

// Two products of which neither reads what the other writes, each with memory of its own for its parts.
bool go_together(const LinearProduct& a, const LinearProduct& b) {
    return a.dtype == SXCUDA_F32 && a.plan.tile_m == 64 && b.plan.tile_m == 64;
}
void launch_together(const LinearProduct (&p)[2], cudaStream_t s) {
    const LinearProducts<2> of = products_of(p);
    const auto kernel = linear_kernel<64, 2>;
    SX_LAUNCH(kernel, static_cast<unsigned>(p[0].plan.workers + p[1].plan.workers), kThreads<64>, 0, s, of);
    launch_join<float>(of, s);
}

// ---- a few rows ----
// A warp has an output feature: its lanes go along the weight's row, V values at a time, and each of up to ROWS
// rows of x has a sum. The weight is read once, by as many warps as there are features; a product on the tensor
// cores needs its parts of K joined to read it as widely. 1024 -> 4096 features, this and the tiles, in us: bf16
// 1 row 3.4 and 12, 4 rows 5.2 and 12, 8 rows 9.3 and 9.5 (4096 -> 4096: 24 and 18); float32 1 row 3.7 and 23, 8
// rows 11 and 24.
constexpr int few_rows_of(int32_t dtype) { return dtype == SXCUDA_F32 ? 8 : 4; }
template <typename T, int V, int ROWS>
__global__ void __launch_bounds__(128) linear_few_kernel(const __grid_constant__ LinearProduct p) {
    const int lane = threadIdx.x & 31;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (n >= p.n) return;
    const T* w = static_cast<const T*>(p.b.data) + n * p.b.stride;
    float sum[ROWS] = {};
#pragma unroll 4
    for (int64_t k = lane * V; k < p.k; k += 32 * V) {
        const auto v = *reinterpret_cast<const Pack<T, V>*>(w + k);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const auto x = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(p.a.data) + (r < p.m ? r : 0) * p.a.stride + k);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[r] = fmaf(to_f32(v.v[i]), to_f32(x.v[i]), sum[r]);
        }
    }
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int o = 16; o; o >>= 1) sum[r] += __shfl_xor_sync(kFullMask, sum[r], o);
        if (lane == r) mine = sum[r];
    }
    if (lane >= p.m) return;
    float z[1] = {mine}, bias[1] = {linear_param(p.bias, p.bias_dtype, n)};
    linear_finish<T, 1>(p, lane, n, z, bias, 1);
}
template <typename T>
void launch_few(const LinearProduct& p, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const auto run = [&](auto kernel) { SX_LAUNCH(kernel, blocks_for(p.n, 4), 128, 0, s, p); };
    const auto rows = [&](auto v) {
        constexpr int N = decltype(v)::value;
        if (p.m == 1) run(linear_few_kernel<T, N, 1>);
        else if (p.m == 2) run(linear_few_kernel<T, N, 2>);
        else if (p.m <= 4) run(linear_few_kernel<T, N, 4>);
        else if constexpr (sizeof(T) == 4) run(linear_few_kernel<T, N, 8>);
    };
    if (p.k % V == 0 && linear_wide(p.a, sizeof(T)) && linear_wide(p.b, sizeof(T))) rows(std::integral_constant<int, V>{});
    else rows(std::integral_constant<int, 1>{});
}

// ---- rows that tensor maps do not take, copied to rows that they do ----
__global__ void __launch_bounds__(256) linear_pack_kernel(const uint16_t* from, int64_t stride, int64_t rows, int32_t cols, uint16_t* to,
                                                          int32_t pitch) {
    const int64_t pieces = pitch / 8, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = i / pieces;
    const int32_t c = static_cast<int32_t>(i - row * pieces) * 8;
    if (row >= rows) return;
    Pack<uint16_t, 8> x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x.v[j] = c + j < cols ? from[row * stride + c + j] : 0;
    *reinterpret_cast<Pack<uint16_t, 8>*>(to + row * pitch + c) = x;
}
int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }

// A matrix of the call as the products read it: itself, or its copy at `at` in the workspace.
struct Matrix {
    const void* data;
    int64_t stride, rows, cols;
    bool copied(int32_t dtype) const { return dtype != SXCUDA_F32 && !linear_tc_takes(data, stride, rows); }
    size_t bytes(int32_t dtype) const { return copied(dtype) ? aligned_bytes(static_cast<size_t>(rows) * pitch_of(cols) * 2) : 0; }
    static size_t aligned_bytes(size_t n) { return (n + 255) / 256 * 256; }
    Matrix ready(int32_t dtype, uint8_t* at, cudaStream_t s) const {
        if (!copied(dtype)) return *this;
        const int64_t pitch = pitch_of(cols);
        SX_LAUNCH(linear_pack_kernel, blocks_for(rows * (pitch / 8), 256), 256, 0, s, static_cast<const uint16_t*>(data), stride, rows,
                  static_cast<int32_t>(cols), reinterpret_cast<uint16_t*>(at), static_cast<int32_t>(pitch));
        return {at, pitch, rows, cols};
    }
    LinearOperand along_k() const { return {data, stride, false}; }  // its rows are the operand's
    LinearOperand across_k() const { return {data, stride, true}; }  // its columns are
};

__device__ __forceinline__ void linear_param_to(void* w, int32_t dtype, int64_t i, float x) {
    if (dtype == SXCUDA_F32) static_cast<float*>(w)[i] = x;
    else if (dtype == SXCUDA_F16) static_cast<__half*>(w)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(x);
}

// ---- v_z = v_y act'(pre), and the sum of its rows ----
// v_z is rounded to the element type, as the tensor cores take it: the gradients of x and of the weight behind an activation
// are then off by 0.0023 of their size in bfloat16 where a v_z of 32 bits leaves 0.0017 (float16 an eighth of both). Two
// 16-bit parts of it would double both products. The bias' sum takes it before the rounding.
// A CTA has 32 V columns (a warp's lanes V each) and a slice of the rows, which its warps take in turn; the grid
// is what the SMs hold. Bound by memory: gelu over bf16 32768 x 4096 163 us (4.9 TB/s); several rows asked for
// at once by a warp, with fewer warps, were slower (2 rows 185 us, 4 rows 222 us).
constexpr int kSlopeWarps = 8, kSlopePerSm = 6;
struct SlopeArgs {
    const void* v_y;
    const void* pre;
    void* v_z;    // NULL: v_y itself
    float* sums;  // [slices, cols] or NULL
    void* v_bias;  // written by the only slice there is, else NULL
    int64_t v_y_stride, pre_stride, v_z_stride, rows, cols, slice;
    int32_t act, bias_dtype;
};
template <typename T, int V>
__global__ void __launch_bounds__(kSlopeWarps * 32, kSlopePerSm) linear_slope_kernel(const SlopeArgs a) {
    __shared__ float part[kSlopeWarps][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * V;
    const int64_t r0 = blockIdx.y * a.slice, r1 = min(r0 + a.slice, a.rows);
    float sum[V] = {};
    if (c < a.cols)
        for (int64_t r = r0 + warp; r < r1; r += kSlopeWarps) {
            const auto g = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.v_y) + r * a.v_y_stride + c);
            Pack<T, V> z{}, to;
            if (a.pre) z = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.pre) + r * a.pre_stride + c);
            float x[V], at[V];
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = to_f32(g.v[i]), at[i] = to_f32(z.v[i]);
            if (a.pre) times_slopes<T>(a.act, at, x);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] += x[i], to.v[i] = from_f32<T>(x[i]);
            if (a.v_z) *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.v_z) + r * a.v_z_stride + c) = to;
        }
    if (!a.sums && !a.v_bias) return;
#pragma unroll
    for (int i = 0; i < V; ++i) part[warp][lane * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += kSlopeWarps * 32) {
        const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 * V + i;
        float x = 0.f;
        for (int w = 0; w < kSlopeWarps; ++w) x += part[w][i];
        if (col >= a.cols) continue;
        if (a.v_bias) linear_param_to(a.v_bias, a.bias_dtype, col, x);
        else a.sums[blockIdx.y * a.cols + col] = x;
    }
}
// Adds the slices' sums of 32 columns: warp w takes every 32nd slice, eight in flight, then the warps are
// added in order.
__global__ void __launch_bounds__(1024) linear_bias_kernel(const float* part, int64_t slices, int64_t cols, void* v_bias, int32_t dtype) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s = 0.f;
    if (c < cols)
        for (int64_t r = warp; r < slices; r += 8 * 32) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = r + i * 32 < slices ? part[(r + i * 32) * cols + c] : 0.f;
            s += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
    sums[warp][lane] = s;
    __syncthreads();
    s = sums[lane][warp];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + warp;
    if (lane || at >= cols) return;
    linear_param_to(v_bias, dtype, at, s);
}

struct SlopePlan {
    int v;
    int64_t strips, slices, slice;
};
SlopePlan slope_plan(const SxLinearInputs& in, const SxLinearGradsIn& g) {
    const int64_t size = dtype_bytes(in.dtype), most = 16 / size;
    const auto wide = [&](const void* p, int64_t stride) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (in.rows <= 1 || stride % most == 0);
    };
    SlopePlan p;
    p.v = in.out_features % most == 0 && wide(g.v_y, g.v_y_stride) && wide(g.pre, g.pre_stride) ? static_cast<int>(most) : 1;
    p.strips = (in.out_features + 32 * p.v - 1) / (32 * p.v);
    const int64_t want = std::max<int64_t>(static_cast<int64_t>(sm_count()) * kSlopePerSm / p.strips, 1);
    p.slice = std::max<int64_t>((in.rows + want - 1) / want, 4 * kSlopeWarps);
    // few: no second kernel (us in one slice and in several: 128 x 2560 gelu 13.2 and 8, without an activation 4.9 and 6)
    if (in.rows <= (g.pre ? 8 : 16) * kSlopeWarps) p.slice = in.rows;
    p.slices = (in.rows + p.slice - 1) / p.slice;
    return p;
}

// The backward's workspace: v_z where it is not v_y, copies of x and weight, the bias' sums, the products' parts.
struct BwdSpace {
    Matrix x, weight, v_y;
    bool v_z = false;  // made
    size_t x_at = 0, weight_at = 0, v_z_at = 0, sums_at = 0, parts_at[2] = {}, bytes = 0;
    BwdSpace(const SxLinearInputs& in, const SxLinearGradsIn& g, const SxLinearGrads& out)
        : x{in.x, in.x_stride, in.rows, in.in_features}, weight{in.weight, in.weight_stride, in.out_features, in.in_features},
          v_y{g.v_y, g.v_y_stride, in.rows, in.out_features} {
        if (in.rows == 0) return;
        const auto take = [&](size_t& at, size_t n) {
            at = bytes;
            bytes += Matrix::aligned_bytes(n);
        };
        v_z = g.pre || ((out.v_x || out.v_weight) && v_y.copied(in.dtype));
        if (v_z) take(v_z_at, static_cast<size_t>(in.rows) * pitch_of(in.out_features) * dtype_bytes(in.dtype));
        if (out.v_weight) take(x_at, x.bytes(in.dtype));
        if (out.v_x) take(weight_at, weight.bytes(in.dtype));
        if (out.v_bias) take(sums_at, static_cast<size_t>(slope_plan(in, g).slices) * in.out_features * 4);
        if (out.v_x) take(parts_at[0], product_plan(in.dtype, in.rows, in.in_features, in.out_features).workspace());
        if (out.v_weight) take(parts_at[1], product_plan(in.dtype, in.out_features, in.in_features, in.rows).workspace());
    }
};

bool few_rows(const SxLinearInputs& in) { return in.rows <= few_rows_of(in.dtype); }

}  // namespace

size_t linear_fwd_workspace(const SxLinearInputs& in) {
    if (in.rows == 0 || few_rows(in)) return 0;
    const Matrix x{in.x, in.x_stride, in.rows, in.in_features}, w{in.weight, in.weight_stride, in.out_features, in.in_features};
    return x.bytes(in.dtype) + w.bytes(in.dtype) + product_plan(in.dtype, in.rows, in.out_features, in.in_features).workspace();
}

void launch_linear_fwd(const SxLinearInputs& in, const SxLinearOutputs& out, void* ws, cudaStream_t s) {
    if (in.rows == 0) return;
    uint8_t* at = static_cast<uint8_t*>(ws);
    const Matrix x{in.x, in.x_stride, in.rows, in.in_features}, w{in.weight, in.weight_stride, in.out_features, in.in_features};
    const bool few = few_rows(in);
    LinearProduct p{};
    p.a = (few ? x : x.ready(in.dtype, at, s)).along_k();
    p.b = (few ? w : w.ready(in.dtype, at += x.bytes(in.dtype), s)).along_k();
    p.m = in.rows, p.n = in.out_features, p.k = in.in_features;
    p.dtype = in.dtype, p.bias_dtype = in.bias_dtype, p.act = in.activation;
    p.bias = in.bias;
    p.residual = out.residual, p.residual_stride = out.residual_stride;
    p.y = out.y, p.y_stride = out.y_stride;
    p.pre = out.pre, p.pre_stride = out.pre_stride;
    if (few) {
        by_dtype(in.dtype, [&](auto t) { launch_few<decltype(t)>(p, s); });
        return;
    }
    p.parts = reinterpret_cast<float*>(at + w.bytes(in.dtype));
    p.plan = product_plan(in.dtype, p.m, p.n, p.k);
    launch_product(p, s);
}

size_t linear_bwd_workspace(const SxLinearInputs& in, const SxLinearGradsIn& g, const SxLinearGrads& out) {
    return BwdSpace(in, g, out).bytes;
}

void launch_linear_bwd(const SxLinearInputs& in, const SxLinearGradsIn& g, const SxLinearGrads& out, void* ws, cudaStream_t s) {
    const int64_t size = dtype_bytes(in.dtype);
    if (in.rows == 0) {
        if (out.v_weight)
            cuda_check(cudaMemset2DAsync(out.v_weight, out.v_weight_stride * size, 0, in.in_features * size, in.out_features, s), "linear_bwd");
        if (out.v_bias) cuda_check(cudaMemsetAsync(out.v_bias, 0, in.out_features * dtype_bytes(in.bias_dtype), s), "linear_bwd");
        return;
    }
    const BwdSpace space(in, g, out);
    uint8_t* at = static_cast<uint8_t*>(ws);
    Matrix v_z = space.v_y;
    if (space.v_z || out.v_bias) {
        const SlopePlan plan = slope_plan(in, g);
        SlopeArgs a{g.v_y, g.pre, nullptr, nullptr, nullptr, g.v_y_stride, g.pre_stride, pitch_of(in.out_features), in.rows, in.out_features, plan.slice, in.activation, in.bias_dtype};
        if (space.v_z) v_z = {a.v_z = at + space.v_z_at, a.v_z_stride, in.rows, in.out_features};
        if (out.v_bias && plan.slices > 1) a.sums = reinterpret_cast<float*>(at + space.sums_at);
        else a.v_bias = out.v_bias;
        by_dtype(in.dtype, [&](auto t) {
            using T = decltype(t);
            const auto kernel = plan.v == 1 ? linear_slope_kernel<T, 1> : linear_slope_kernel<T, 16 / sizeof(T)>;
            SX_LAUNCH(kernel, dim3(static_cast<unsigned>(plan.strips), static_cast<unsigned>(plan.slices)), kSlopeWarps * 32, 0, s, a);
        });
        if (a.sums)
            SX_LAUNCH(linear_bias_kernel, blocks_for(in.out_features, 32), 1024, 0, s, a.sums, plan.slices, in.out_features, out.v_bias, in.bias_dtype);
    }
    LinearProduct products[2]{};
    auto& [p, w] = products;
    if (out.v_x) {
        p.a = v_z.along_k();
        p.b = space.weight.ready(in.dtype, at + space.weight_at, s).across_k();
        p.m = in.rows, p.n = in.in_features, p.k = in.out_features;
        p.y = out.v_x, p.y_stride = out.v_x_stride;
    }
    if (out.v_weight) {
        w.a = v_z.across_k();
        w.b = space.x.ready(in.dtype, at + space.x_at, s).across_k();
        w.m = in.out_features, w.n = in.in_features, w.k = in.rows;
        w.y = out.v_weight, w.y_stride = out.v_weight_stride;
    }
    for (LinearProduct& each : products) {
        if (!each.y) continue;
        each.dtype = in.dtype;
        each.parts = reinterpret_cast<float*>(at + space.parts_at[&each - products]);
        each.plan = product_plan(in.dtype, each.m, each.n, each.k);
    }
    if (p.y && w.y && go_together(p, w)) {
        launch_together(products, s);
        return;
    }
    for (const LinearProduct& each : products)
        if (each.y) launch_product(each, s);
}

}  // namespace sx
