// The translation unit of the fine-tuning operators: their kernel templates are instantiated here,
// next to their host launchers (variant choice, launch shape, PDL attribute).
#include "train.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>
#include <utility>

#include "adamw.cuh"
#include "launch.h"
#include "linear_small.cuh"
#include "linear_tc.cuh"
#include "loss.cuh"
#include "norm.cuh"

namespace jc {

static int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess) return sms;
    const int k = known[dev & 63].load();
    if (k > 0) return k;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev & 63].store(sms);
    return sms;
}

// Blocks of a kernel that an SM holds (asked once: the kernels run on one architecture).
template <class K>
static bool blocks_per_sm(K kern, int threads, int smem, std::atomic<int> &known, int *n) {
    *n = known.load();
    if (*n > 0) return true;
    if (!cuda_ok(cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kern, threads, (size_t)smem), "occupancy")) return false;
    if (*n <= 0) {
        set_error("a kernel does not fit an SM");
        return false;
    }
    known.store(*n);
    return true;
}

static bool aligned16(const void *p, size_t ld, size_t size) {
    return (reinterpret_cast<uintptr_t>(p) | (ld * size)) % 16 == 0;
}

// ---------------------------------------------------------------------------------------------
// layer norm

// Calls f<T>() for an element type.
template <class F>
static bool with_type(uint32_t type, F &&f) {
    if (type == JC_F16) return f(__half());
    if (type == JC_BF16) return f(__nv_bfloat16());
    return f(float());
}

template <int N>
using Int = std::integral_constant<int, N>;

// The group that holds a row of d elements: the smallest G x E that does (a warp up to 1024, so
// that no reduction crosses warps, then four to sixteen).
template <class F>
static bool with_group(uint32_t d, F &&f) {
    if (d <= 256) return f(Int<32>(), Int<8>());
    if (d <= 512) return f(Int<32>(), Int<16>());
    if (d <= 768) return f(Int<32>(), Int<24>());
    if (d <= 1024) return f(Int<32>(), Int<32>());
    if (d <= 2048) return f(Int<128>(), Int<16>());
    if (d <= 4096) return f(Int<128>(), Int<32>());
    if (d <= 8192) return f(Int<256>(), Int<32>());
    return f(Int<512>(), Int<32>());
}

// How a layer norm's tensors are read. All rows that start alike (the same remainder by 16 bytes in
// every tensor, row for row) are read in 16-byte chunks; the others element by element.
struct NormLayout {
    bool chunks = true;
    uint32_t period = 1;  // rows this far apart start alike
    uint32_t span;        // the elements a row's chunks hold
};

static NormLayout norm_layout(uint32_t d, size_t size, std::initializer_list<std::pair<const void *, size_t>> ts) {
    NormLayout l;
    const uint32_t v = (uint32_t)(16 / size);
    const auto [p0, ld0] = *ts.begin();
    bool aligned = true;
    for (const auto &[p, ld] : ts) {
        if (!p) continue;
        if ((reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(p0)) % 16 || (ld - ld0) * size % 16) l.chunks = false;
        if (!aligned16(p, ld, size)) aligned = false;
    }
    l.period = l.chunks && !aligned ? v : 1;
    l.span = l.period > 1 ? d + v - 1 : d;
    if (l.span > NORM_MAX_D) {
        l.chunks = false;
        l.period = 1;
        l.span = d;
    }
    return l;
}

// A multiple of `period` blocks, enough for `groups` rows each but no more than `most`.
static uint32_t norm_blocks(uint32_t rows, uint32_t groups, uint32_t period, uint32_t most) {
    const uint32_t per = (rows + period - 1) / period;  // rows of a class
    return std::min((per + groups - 1) / groups, most / period) * period;
}

bool launch_norm(const NormArgs &a, cudaStream_t s) {
    if (a.rows == 0) return true;
    unsigned int *err = module_error_word();
    if (!err) return false;
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        const NormLayout l = norm_layout(a.d, sizeof(T), {{a.x, a.ldx}, {a.y, a.ldy}});
        return with_group(l.span, [&](auto g, auto e) {
            constexpr int G = g, E = e;
            const NormParams p{a.x, a.ldx, a.gamma, a.beta, a.eps, a.rows, a.d, l.period, a.y, a.ldy, a.stats, err};
            auto go = [&](auto kern, std::atomic<uint64_t> &set, std::atomic<int> &resident, auto shape) {
                using S = decltype(shape);
                int per_sm = 0;
                if (!ensure_smem(kern, S::SMEM, set) || !blocks_per_sm(kern, S::THREADS, S::SMEM, resident, &per_sm))
                    return false;
                const dim3 grid(norm_blocks(a.rows, S::GROUPS * S::ROWS, l.period, (uint32_t)(sm_count() * per_sm)));
                return launch_ex(kern, grid, dim3(S::THREADS), S::SMEM, s, true, "layer_norm", p);
            };
            static std::atomic<uint64_t> set_v{0}, set_1{0};
            static std::atomic<int> res_v{0}, res_1{0};
            return l.chunks ? go(norm_kernel<T, VEC<T>, G, E>, set_v, res_v, NormShape<T, VEC<T>, G, E>())
                            : go(norm_kernel<T, 1, G, E>, set_1, res_1, NormShape<T, 1, G, E>());
        });
    });
}

// Blocks of the backward kernel at most: one a SM. Each leaves a row of partial sums (up to seven
// blocks more than rows: a multiple of the period).
constexpr uint32_t NORM_BWD_BLOCKS = 148;

// A few rows take one block, which then writes dgamma and dbeta without a second kernel: 3 us less
// of launches than it costs to have a group take NORM_BWD_ALONE rows one after the other.
constexpr uint32_t NORM_BWD_ALONE = 8;

size_t norm_bwd_ws_floats(uint32_t rows, uint32_t d) {
    return rows > NORM_BWD_ALONE ? std::min<size_t>((size_t)rows + 7, NORM_BWD_BLOCKS) * 2 * d : 0;
}

static bool launch_column_sum(const float *ws, uint32_t parts, uint32_t n, uint32_t columns, float *a,
                              float *b, cudaStream_t s) {
    return launch_ex(column_sum_kernel, dim3((columns + 31) / 32), dim3(1024), 0, s, true, "column sums", ws,
                     parts, n, columns, a, b);
}

bool launch_norm_bwd(const NormBwdArgs &a, cudaStream_t s) {
    const bool sums = a.dgamma || a.dbeta;
    uint32_t blocks = 0;
    unsigned int *err = module_error_word();
    if (!err) return false;
    if (a.rows > 0) {
        const bool ok = with_type(a.type, [&](auto t) {
            using T = decltype(t);
            NormLayout l = norm_layout(a.d, sizeof(T), {{a.x, a.ldx}, {a.dy, a.lddy}, {a.dx, a.lddx}, {a.add, a.ldadd}});
            if (a.rows <= NORM_BWD_ALONE && l.period > 1) l = NormLayout{false, 1, a.d};  // one class of rows only
            return with_group(l.span, [&](auto g, auto e) {
                constexpr int G = g, E = e;
                const NormBwdParams p{a.dy, a.lddy, a.x, a.ldx, a.gamma, a.stats, a.add, a.ldadd, a.rows,
                                      a.d, l.period, a.dx, a.lddx, a.ws, a.dgamma, a.dbeta, err};
                auto go = [&](auto kern, std::atomic<uint64_t> &set, auto shape) {
                    using S = decltype(shape);
                    blocks = a.rows <= NORM_BWD_ALONE ? 1 : norm_blocks(a.rows, S::GROUPS, l.period, NORM_BWD_BLOCKS);
                    return ensure_smem(kern, S::SMEM, set) &&
                           launch_ex(kern, dim3(blocks), dim3(S::THREADS), S::SMEM, s, true, "layer_norm_backward", p);
                };
                static std::atomic<uint64_t> set_v{0}, set_1{0};
                return l.chunks ? go(norm_bwd_kernel<T, VEC<T>, G, E>, set_v, NormBwdShape<T, VEC<T>, G, E>())
                                : go(norm_bwd_kernel<T, 1, G, E>, set_1, NormBwdShape<T, 1, G, E>());
            });
        });
        if (!ok) return false;
    }
    return !sums || blocks == 1 || launch_column_sum(a.ws, blocks, a.d, 2 * a.d, a.dgamma, a.dbeta, s);
}

// ---------------------------------------------------------------------------------------------
// linear

template <class F>
static bool with_half(uint32_t type, F &&f) {
    return type == JC_F16 ? f(__half()) : f(__nv_bfloat16());
}

template <class F>
static bool with_act(uint32_t act, F &&f) {
    if (act == JC_EPI_RELU) return f(std::integral_constant<uint32_t, JC_EPI_RELU>());
    if (act == JC_EPI_GELU) return f(std::integral_constant<uint32_t, JC_EPI_GELU>());
    return f(std::integral_constant<uint32_t, 0>());
}

// One product c = a b^T and how it is run.
struct Product {
    LinearOperand a{}, b{};  // the contiguous axis of each has stride 1
    uint32_t m = 0, n = 0, k = 0, act = 0;
    const float *bias = nullptr;
    const void *res = nullptr;
    size_t ldres = 0;
    void *c = nullptr;
    size_t ldc = 0;
    void *z = nullptr;
    size_t ldz = 0;
    float *ws = nullptr;
    uint32_t splits = 1;
};

// The tensor map of an operand: boxes of 64 contracted elements x `rows` rows where the contracted
// axis is contiguous, else of 64 x 64.
template <class T>
static bool make_operand_map(CUtensorMap *map, const LinearOperand &o, uint32_t rows, uint32_t k, bool mn,
                             uint32_t box_rows) {
    auto fn = encode_fn();
    if (!fn) {
        set_error("cuTensorMapEncodeTiled is not available from the CUDA driver");
        return false;
    }
    cuuint64_t dims[2] = {mn ? rows : k, mn ? k : rows};
    cuuint64_t strides[1] = {(mn ? o.sk : o.si) * 2};
    cuuint32_t box[2] = {64, mn ? 64 : box_rows}, es[2] = {1, 1};
    const CUresult r =
        fn(map, std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
           2, const_cast<void *>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return true;
    set_error("linear: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return false;
}

// Whether TMA can load a matrix: its rows on 16-byte boundaries (and a row distance it can hold).
static bool tma_ok(const void *p, size_t ld) { return aligned16(p, ld, 2) && ld * 2 < ((size_t)1 << 40); }

static size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// A matrix argument's copy for TMA, if it needs one: where in the workspace, and how long.
struct Pad {
    bool need = false;
    size_t at = 0, ld = 0, bytes = 0;
};
static Pad plan_pad(const void *p, size_t ld, uint32_t rows, uint32_t cols, size_t at) {
    Pad d;
    d.need = p && !tma_ok(p, ld);
    d.at = at;
    d.ld = round_up(cols, 8);
    d.bytes = d.need ? round_up((size_t)rows * d.ld * 2, 256) : 0;
    return d;
}

// Queues the copies of two matrices that need them and points the arguments at them.
static bool launch_pads(uint8_t *ws, const Pad &a, const void **pa, size_t *lda, uint32_t rows_a, uint32_t cols_a,
                        const Pad &b, const void **pb, size_t *ldb, uint32_t rows_b, uint32_t cols_b, cudaStream_t s) {
    PadParams p{};
    uint32_t blocks[2] = {0, 0};
    auto add = [&](int i, const Pad &d, const void **src, size_t *ld, uint32_t rows, uint32_t cols) {
        if (!d.need || rows == 0) return;
        p.src[i] = static_cast<const uint16_t *>(*src);
        p.ld[i] = *ld;
        p.rows[i] = rows;
        p.cols[i] = cols;
        p.dst[i] = reinterpret_cast<uint16_t *>(ws + d.at);
        p.ldd[i] = d.ld;
        blocks[i] = (uint32_t)std::min<uint64_t>(((uint64_t)rows * (d.ld / 8) + 255) / 256, 148 * 16);
        *src = ws + d.at;
        *ld = d.ld;
    };
    add(0, a, pa, lda, rows_a, cols_a);
    add(1, b, pb, ldb, rows_b, cols_b);
    p.first = blocks[0];
    if (blocks[0] + blocks[1] == 0) return true;
    return launch_ex(linear_pad_kernel, dim3(blocks[0] + blocks[1]), dim3(256), 0, s, true, "linear", p);
}

static bool out_vec(const Product &q) {
    return q.n % 8 == 0 && aligned16(q.c, q.ldc, 2) && (!q.z || aligned16(q.z, q.ldz, 2)) &&
           (!q.res || aligned16(q.res, q.ldres, 2));
}

// Runs the forward product (q[0]) or (GRADS) dw's and dx's, either of which may be without rows.
template <class T, int BN, int CTAS, bool GRADS, uint32_t ACT, bool VEC>
static bool launch_tc(const Product *q, cudaStream_t s) {
    static std::atomic<uint64_t> smem_set{0};
    auto kern = linear_tc_kernel<T, BN, CTAS, GRADS, ACT, VEC>;
    LinearTcKernelParams kp{};
    kp.err = module_error_word();
    using Mem = LtTcSmem<BN, CTAS>;
    if (!kp.err || !ensure_smem(kern, Mem::BYTES, smem_set)) return false;
    uint64_t items = 0;
    for (int w = 0; w < (GRADS ? 2 : 1); w++) {
        const Product &r = q[w];
        if (r.m == 0) continue;
        const uint32_t tiles_m = (r.m + CTAS * LT_BM - 1) / (CTAS * LT_BM), tiles_n = (r.n + BN - 1) / BN;
        const uint64_t mine = (uint64_t)tiles_m * tiles_n * r.splits;
        items += mine;
        if (items > 0x7FFFFFFFull) {
            set_error("linear: too many tiles");
            return false;
        }
        kp.items[w] = (uint32_t)mine;
        kp.p[w] = LinearTcParams{r.m,     r.n, r.k,   r.bias, r.res, r.ldres,  r.c,     r.ldc,
                                 r.z,     r.ldz, r.ws, r.splits, tiles_m, tiles_n};
        if (!make_operand_map<T>(&kp.map_a[w], r.a, r.m, r.k, GRADS && w == 0, LT_BM) ||
            !make_operand_map<T>(&kp.map_b[w], r.b, r.n, r.k, GRADS, BN / CTAS))
            return false;
    }
    if constexpr (CTAS == 1) {
        const uint32_t grid = (uint32_t)std::min<uint64_t>(items, (uint64_t)sm_count());
        return launch_ex(kern, dim3(grid), dim3(LT_TC_THREADS), Mem::BYTES, s, true, "linear", kp);
    } else {
        static std::atomic<int> max_pairs{0};
        int pairs = max_pairs.load();
        if (pairs == 0) {
            if (!max_clusters(kern, 2, LT_TC_THREADS, Mem::BYTES, &pairs)) return false;
            max_pairs.store(pairs);
        }
        const uint32_t grid = 2 * (uint32_t)std::min<uint64_t>(items, (uint64_t)pairs);
        return launch_ex_cluster(kern, dim3(grid), dim3(LT_TC_THREADS), Mem::BYTES, s, true, dim3(2, 1, 1), "linear", kp);
    }
}

// How the TMA kernel tiles a product: `ctas` x 128 rows by bn columns.
struct Tiling {
    uint32_t ctas, bn;
};
constexpr Tiling TILINGS[] = {{1, 64}, {1, 128}, {2, 128}, {2, 256}};

// An item's microseconds: about 0.36 us per 64 contracted elements (one thread's MMAs complete in order at
// about 130 cycles each whatever their width; the clock under load is what it is), and 0.5 us.
struct Items {
    uint64_t count = 0;
    double us = 0.0;
};
static Items tc_items(uint32_t m, uint32_t n, uint32_t k, Tiling t, uint32_t splits) {
    if (m == 0) return {};
    const uint32_t rows = t.ctas * LT_BM, blocks = ((k + LT_BK - 1) / LT_BK + splits - 1) / splits;
    return {(uint64_t)((m + rows - 1) / rows) * ((n + t.bn - 1) / t.bn) * splits, 0.36 * blocks + 0.5};
}

// Microseconds of a launch of two kinds of items: whole rounds of each (dw's items spread over the units
// beside dx's cost more than the sum of the work says: at 12288 x 768 x 2048 two splits, 48 items beside
// dx's 144, take 138 us, three, 72 items for 74 pairs, 98), then the first loads and the last epilogue.
static double tc_us(Items a, Items b, Tiling t, uint32_t sms) {
    const uint32_t units = sms / t.ctas;
    return (double)((a.count + units - 1) / units) * a.us + (double)((b.count + units - 1) / units) * b.us + 2.0 +
           0.008 * t.bn;
}

// Runs products with a tiling.
template <class T, bool GRADS, uint32_t ACT>
static bool launch_products(const Product *q, Tiling t, cudaStream_t s) {
    bool vec = true;
    for (int w = 0; w < (GRADS ? 2 : 1); w++) vec = vec && (q[w].m == 0 || out_vec(q[w]));
    auto run = [&](auto c, auto w) {
        constexpr int CTAS = decltype(c)::value, BN = decltype(w)::value;
        return vec ? launch_tc<T, BN, CTAS, GRADS, ACT, true>(q, s) : launch_tc<T, BN, CTAS, GRADS, ACT, false>(q, s);
    };
    if (t.ctas == 2) return t.bn == 256 ? run(Int<2>(), Int<256>()) : run(Int<2>(), Int<128>());
    return t.bn == 128 ? run(Int<1>(), Int<128>()) : run(Int<1>(), Int<64>());
}

// Calls f(N) for the smallest instantiated number of columns a thin layer of n has.
template <class F>
static bool with_thin(uint32_t n, F &&f) {
    if (n <= 1) return f(Int<1>());
    if (n <= 2) return f(Int<2>());
    if (n <= 4) return f(Int<4>());
    return f(Int<8>());
}

static Tiling forward_tiling(uint32_t m, uint32_t n, uint32_t k, double *us) {
    Tiling best = TILINGS[0];
    *us = 1e30;
    for (const Tiling &t : TILINGS) {
        const double v = tc_us(tc_items(m, n, k, t, 1), {}, t, (uint32_t)sm_count());
        if (v > *us) continue;
        best = t;
        *us = v;
    }
    return best;
}

// Whether few rows go to linear_rows_kernel, which reads the weights once for 16 of them: 1.8 us and 0.55
// for a million products of 16 rows (384 x 768: 1.9 us at 16 rows, 3.4 at 128; 2304 x 768: 5.3 at 64, 8.7
// at 128), where the tensor tiles of 128 rows take what tc_us says less a fifth when they are few (384 x
// 768 5.6 to 5.9 us, 2304 x 768 5.8 to 6.0, 768 x 2048 11.2 to 11.5 against 5.9 and 8.1 at 64 and 128).
static bool few_rows(uint32_t m, uint32_t n, uint32_t k, double tc) {
    const uint32_t groups = (m + 15) / 16;
    return groups <= 65535 && 1.8 + 0.55e-6 * groups * (double)n * k < 0.8 * tc;
}

bool launch_linear(const LinearArgs &a, cudaStream_t s) {
    if (a.m == 0) return true;
    const LinearRowsParams rp{a.x, a.ldx, a.w, a.ldw, a.bias, a.res, a.ldres, a.y, a.ldy, a.z, a.ldz, a.m, a.n, a.k};
    const bool vec = a.k % 8 == 0 && aligned16(a.x, a.ldx, 2) && aligned16(a.w, a.ldw, 2);
    if (a.n <= LTHIN_MAX)
        return with_half(a.type, [&](auto t) {
            using T = decltype(t);
            return with_act(a.act, [&](auto act) {
                return with_thin(a.n, [&](auto n) {
                    constexpr uint32_t ACT = decltype(act)::value;
                    constexpr int N = decltype(n)::value;
                    const dim3 grid((a.m + 8 * LTHIN_ROWS - 1) / (8 * LTHIN_ROWS));
                    return vec ? launch_ex(linear_thin_kernel<T, N, true, ACT>, grid, dim3(256), 0, s, true, "linear", rp)
                               : launch_ex(linear_thin_kernel<T, N, false, ACT>, grid, dim3(256), 0, s, true, "linear", rp);
                });
            });
        });
    double tc = 0.0;
    const Tiling tiling = forward_tiling(a.m, a.n, a.k, &tc);
    if (few_rows(a.m, a.n, a.k, tc))
        return with_half(a.type, [&](auto t) {
            return with_act(a.act, [&](auto act) {
                using T = decltype(t);
                constexpr uint32_t ACT = decltype(act)::value;
                const dim3 grid((a.n + 7) / 8, (a.m + 15) / 16);
                return vec ? launch_ex(linear_rows_kernel<T, ACT, true>, grid, dim3(32 * LR_WARPS), 0, s, true, "linear", rp)
                           : launch_ex(linear_rows_kernel<T, ACT, false>, grid, dim3(32 * LR_WARPS), 0, s, true, "linear", rp);
            });
        });
    const void *x = a.x, *w = a.w;
    size_t ldx = a.ldx, ldw = a.ldw;
    const Pad px = plan_pad(x, ldx, a.m, a.k, 0), pw = plan_pad(w, ldw, a.n, a.k, px.bytes);
    if (!launch_pads(static_cast<uint8_t *>(a.ws), px, &x, &ldx, a.m, a.k, pw, &w, &ldw, a.n, a.k, s)) return false;
    Product q;
    q.a = LinearOperand{x, ldx, 1};
    q.b = LinearOperand{w, ldw, 1};
    q.m = a.m;
    q.n = a.n;
    q.k = a.k;
    q.bias = a.bias;
    q.res = a.res;
    q.ldres = a.ldres;
    q.c = a.y;
    q.ldc = a.ldy;
    q.z = a.z;
    q.ldz = a.ldz;
    return with_half(a.type, [&](auto t) {
        return with_act(a.act, [&](auto act) {
            return launch_products<decltype(t), false, decltype(act)::value>(&q, tiling, s);
        });
    });
}

size_t linear_ws_bytes(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n, uint32_t k) {
    const size_t bytes = plan_pad(x, ldx, m, k, 0).bytes + plan_pad(w, ldw, n, k, 0).bytes;
    if (bytes == 0 || n <= LTHIN_MAX) return 0;
    double tc = 0.0;
    forward_tiling(m, n, k, &tc);
    return few_rows(m, n, k, tc) ? 0 : bytes;
}

// The tiling of both gradients' products and the splits of dw's contraction, which runs over the rows: its
// few tiles are split so that they still fill the SMs. By the shape alone, so that a gradient has the same
// bits whichever others are asked for. The last shape's plan is kept (weighing the choices takes 2 us).
struct GradPlan {
    uint32_t m = 0, n = 0, k = 0, splits = 1;
    Tiling tiling{};
};
static GradPlan plan_grads(uint32_t m, uint32_t n, uint32_t k) {
    static thread_local GradPlan p;
    if (p.m == m && p.n == n && p.k == k && p.tiling.bn) return p;
    p = GradPlan{m, n, k};
    const uint32_t sms = 148, blocks = (m + LT_BK - 1) / LT_BK;
    double best = 1e30;
    for (const Tiling &t : TILINGS)
        for (uint32_t s : {1u, 2u, 3u, 4u, 5u, 6u, 8u, 12u, 16u, 24u, 32u}) {
            if (s > std::max(1u, blocks)) break;
            double us = tc_us(tc_items(n, k, m, t, s), tc_items(m, k, n, t, 1), t, sms);
            if (s > 1) us += 2.0 + 1.2e-6 * s * n * k;  // the partial sums, written and read
            if (us <= best) {
                best = us;
                p.tiling = t;
                p.splits = s;
            }
        }
    return p;
}

// The backward pass's workspace: dz (16 bits, rows padded to 16 bytes), the column sums' parts, dw's
// partial products, the copies of w and x where TMA cannot load them, each from a 256-byte boundary.
struct LinearBwdPlan {
    uint32_t dz_rows, dz_parts, splits;
    uint32_t thin_blocks;  // few columns: blocks along the rows, each with its sums; nothing else used
    size_t lddz, part_at, ws_at, bytes;
    Pad w, x;
    Tiling tiling;
};

static LinearBwdPlan plan_linear_bwd(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n,
                                     uint32_t k) {
    LinearBwdPlan p{};
    auto up = [](size_t v) { return round_up(v, 256); };
    // Rows a block of the dz kernel takes: few rows go to one, which then writes dbias itself; of very many
    // each takes more, as a grid has 65535 blocks along y.
    p.dz_rows = m <= 2 * DZ_ROWS ? 2 * DZ_ROWS : std::max(DZ_ROWS, (m + 65534) / 65535);
    p.dz_parts = (m + p.dz_rows - 1) / p.dz_rows;
    p.lddz = (n + 7) / 8 * 8;
    p.part_at = up((size_t)m * p.lddz * 2);
    p.ws_at = p.part_at + up((size_t)p.dz_parts * n * 4);
    if (n <= LTHIN_MAX && k <= LTHIN_MAX_K) {
        p.thin_blocks = std::max(1u, std::min((m + 31) / 32, 148u * 2));
        p.bytes = up((size_t)p.thin_blocks * ((size_t)n * k + n) * 4);
        return p;
    }
    const GradPlan g = plan_grads(m, n, k);
    p.tiling = g.tiling;
    p.splits = g.splits;
    p.bytes = p.ws_at + (p.splits > 1 ? up((size_t)p.splits * n * k * 4) : 0);
    p.w = plan_pad(w, ldw, n, k, p.bytes);
    p.x = plan_pad(x, ldx, m, k, p.bytes + p.w.bytes);
    p.bytes += p.w.bytes + p.x.bytes;
    return p;
}

size_t linear_bwd_ws_bytes(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n, uint32_t k) {
    return plan_linear_bwd(x, ldx, w, ldw, m, n, k).bytes;
}

static bool launch_linear_thin_bwd(const LinearBwdArgs &a, uint32_t blocks, cudaStream_t s) {
    return with_half(a.type, [&](auto t) {
        using T = decltype(t);
        const bool sums = a.dw || a.dbias;
        float *part = sums ? static_cast<float *>(a.ws) : nullptr;  // without rows there may be none
        if (a.m > 0) {
            const LinearThinBwdParams p{a.dy, a.lddy, a.x, a.ldx, a.w, a.ldw, a.z, a.ldz, a.m, a.n, a.k,
                                        a.dx, a.lddx, part, a.dw != nullptr};
            const bool vec = a.k % 8 == 0 && (!a.dw || aligned16(a.x, a.ldx, 2)) &&
                             (!a.dx || (aligned16(a.w, a.ldw, 2) && aligned16(a.dx, a.lddx, 2)));
            const dim3 grid(blocks, (a.k + 255) / 256);
            if (!with_act(a.act, [&](auto act) {
                    return with_thin(a.n, [&](auto n) {
                        constexpr uint32_t ACT = decltype(act)::value;
                        constexpr int N = decltype(n)::value;
                        return vec ? launch_ex(linear_thin_bwd_kernel<T, N, true, ACT>, grid, dim3(256), 0, s, true, "linear_backward", p)
                                   : launch_ex(linear_thin_bwd_kernel<T, N, false, ACT>, grid, dim3(256), 0, s, true, "linear_backward", p);
                    });
                }))
                return false;
        }
        if (!sums) return true;
        return launch_ex(linear_thin_finish_kernel<T>, dim3((a.n * a.k + a.n + 31) / 32), dim3(1024), 0, s, true,
                         "linear_backward", (const float *)part, a.m ? blocks : 0u, a.n, a.k, static_cast<T *>(a.dw),
                         a.lddw, a.dbias);
    });
}

bool launch_linear_bwd(const LinearBwdArgs &a, cudaStream_t s) {
    const LinearBwdPlan plan = plan_linear_bwd(a.dw ? a.x : nullptr, a.ldx, a.dx ? a.w : nullptr, a.ldw, a.m, a.n, a.k);
    uint8_t *ws = static_cast<uint8_t *>(a.ws);
    if (plan.thin_blocks) return launch_linear_thin_bwd(a, plan.thin_blocks, s);
    float *part = reinterpret_cast<float *>(ws + plan.part_at);
    return with_half(a.type, [&](auto t) {
        using T = decltype(t);
        const void *dz = a.dy;
        size_t lddz = a.lddy;
        // dz is dy itself where there is no activation and TMA can load dy.
        const bool write = (a.dx || a.dw) && (a.act || !aligned16(a.dy, a.lddy, 2));
        if (a.m > 0 && (write || a.dbias)) {
            const DzParams p{a.dy, a.lddy, a.z, a.ldz, a.m, a.n, plan.dz_rows, write ? ws : nullptr, plan.lddz,
                             a.dbias ? (plan.dz_parts == 1 ? a.dbias : part) : nullptr};
            if (write) {
                dz = ws;
                lddz = plan.lddz;
            }
            const bool vec = a.n % 8 == 0 && aligned16(a.dy, a.lddy, 2) && (!a.act || aligned16(a.z, a.ldz, 2));
            const uint32_t cols = vec ? 256 : 32;
            const dim3 grid((a.n + cols - 1) / cols, plan.dz_parts);
            if (!with_act(a.act, [&](auto act) {
                    constexpr uint32_t ACT = decltype(act)::value;
                    return vec ? launch_ex(linear_dz_kernel<T, ACT, 8>, grid, dim3(256), 0, s, true, "dz", p)
                               : launch_ex(linear_dz_kernel<T, ACT, 1>, grid, dim3(256), 0, s, true, "dz", p);
                }))
                return false;
        }
        const void *x = a.x, *w = a.w;
        size_t ldx = a.ldx, ldw = a.ldw;
        if (a.m > 0 && !launch_pads(ws, plan.w, &w, &ldw, a.n, a.k, plan.x, &x, &ldx, a.m, a.k, s)) return false;
        LinearFinishParams f{};
        Product q[2];  // dw, dx
        if (a.dw && a.m > 0) {
            q[0].a = LinearOperand{dz, 1, lddz};
            q[0].b = LinearOperand{x, 1, ldx};
            q[0].m = a.n;
            q[0].n = a.k;
            q[0].k = a.m;
            q[0].c = a.dw;
            q[0].ldc = a.lddw;
            q[0].splits = plan.splits;
            if (plan.splits > 1) f.ws = q[0].ws = reinterpret_cast<float *>(ws + plan.ws_at);
        }
        if (a.dx && a.m > 0) {
            q[1].a = LinearOperand{dz, lddz, 1};
            q[1].b = LinearOperand{w, 1, ldw};
            q[1].m = a.m;
            q[1].n = a.k;
            q[1].k = a.n;
            q[1].c = a.dx;
            q[1].ldc = a.lddx;
        }
        if ((q[0].m || q[1].m) && !launch_products<T, true, 0>(q, plan.tiling, s)) return false;
        if (a.dw && (f.ws || a.m == 0)) {
            f.splits = a.m ? plan.splits : 0;
            f.m = a.n;
            f.n = a.k;
            f.c = a.dw;
            f.ldc = a.lddw;
        }
        const bool vec = f.n % 8 == 0 && aligned16(f.c, f.ldc, 2);
        const uint64_t threads = (uint64_t)f.m * (vec ? f.n / 8 : f.n);
        f.join_blocks = (uint32_t)std::min<uint64_t>((threads + 255) / 256, 148 * 16);
        if (a.dbias && !(a.m > 0 && plan.dz_parts == 1)) {
            f.part = part;
            f.parts = a.m ? plan.dz_parts : 0;
            f.bias_n = a.n;
            f.dbias = a.dbias;
        }
        const dim3 grid(f.join_blocks + (f.bias_n + 31) / 32);
        if (grid.x == 0) return true;
        return vec ? launch_ex(linear_finish_kernel<T, 8>, grid, dim3(256), 0, s, true, "linear_backward", f)
                   : launch_ex(linear_finish_kernel<T, 1>, grid, dim3(256), 0, s, true, "linear_backward", f);
    });
}

// ---------------------------------------------------------------------------------------------
// loss and optimizer

// Requests of up to this many logits on average go a lane each (a warp's 32 must fit LOSS_SMEM).
constexpr uint32_t LOSS_SHORT = 24;

bool launch_choice_loss(const LossArgs &a, cudaStream_t s) {
    if (a.requests == 0) return true;
    unsigned int *err = module_error_word();
    if (!err) return false;
    const LossParams p{a.logits, a.n_logits, a.offsets, a.gold, a.weight, a.requests, a.loss, a.dlogits, err};
    const uint32_t mean = a.n_logits / a.requests;
    if (mean <= LOSS_SHORT) {
        static std::atomic<int> resident{0};
        int per_sm = 0;
        if (!blocks_per_sm(loss_short_kernel, 32 * LOSS_WARPS, 0, resident, &per_sm)) return false;
        const uint32_t blocks = (a.requests + 32 * LOSS_WARPS - 1) / (32 * LOSS_WARPS);
        return launch_ex(loss_short_kernel, dim3(std::min(blocks, (uint32_t)(sm_count() * per_sm))), dim3(32 * LOSS_WARPS),
                         0, s, true, "choice_loss", p);
    }
    if (mean <= 512) return launch_ex(loss_group_kernel<32>, dim3((a.requests + 3) / 4), dim3(128), 0, s, true, "choice_loss", p);
    return launch_ex(loss_group_kernel<256>, dim3(a.requests), dim3(256), 0, s, true, "choice_loss", p);
}

bool launch_adamw(const AdamwStep &a, cudaStream_t s) {
    if (a.n_chunks == 0) return true;
    AdamwParams p{};
    p.tensors = a.tensors;
    p.chunks = a.chunks;
    p.grad_scale = a.grad_scale;
    p.beta1 = (float)a.beta1;
    p.beta2 = (float)a.beta2;
    p.one_minus_beta1 = (float)(1.0 - a.beta1);
    p.one_minus_beta2 = (float)(1.0 - a.beta2);
    p.lr = a.lr;
    p.eps = a.eps;
    p.minus_zero = -0.0f;
    p.inv_bias1 = (float)(1.0 / (1.0 - std::pow(a.beta1, (double)a.step)));
    p.inv_bias2 = (float)(1.0 / (1.0 - std::pow(a.beta2, (double)a.step)));
    p.n_chunks = a.n_chunks;
    auto go = [&](auto kern, std::atomic<int> &resident) {
        int per_sm = 0;
        if (!blocks_per_sm(kern, ADAMW_THREADS, 0, resident, &per_sm)) return false;
        const uint32_t grid = std::min(a.n_chunks, (uint32_t)(sm_count() * per_sm));
        return launch_ex(kern, dim3(grid), dim3(ADAMW_THREADS), 0, s, true, "adamw", p);
    };
    static std::atomic<int> res_8{0}, res_32{0};
    return a.bits == 8 ? go(adamw_kernel<8>, res_8) : go(adamw_kernel<32>, res_32);
}

}  // namespace jc
