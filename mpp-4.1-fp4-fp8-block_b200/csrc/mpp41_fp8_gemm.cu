// Host side of the FP8 block-scaled products: shape checks, tensor maps, the
// choice of kernel and the launch.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>

#include "mpp41_fp8_gemm.cuh"
#include "mpp41_internal.h"

namespace mpp41 {
namespace fp8 {

namespace {

constexpr int kMaxDevices = 64;

int sm_count(int dev)
{
    static std::atomic<int> n[kMaxDevices];
    int v = n[dev].load(std::memory_order_relaxed);
    if (!v) {
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
        n[dev].store(v, std::memory_order_relaxed);
    }
    return v;
}

template <int BN, int AR, int E, int MODE> cudaError_t prepare(int dev)
{
    static std::atomic<uint64_t> done;
    if (done.load(std::memory_order_acquire) >> dev & 1u) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(fp8_gemm_kernel<BN, AR, E, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(Cfg<BN, AR, MODE>::kSmem + group_bytes(kFp8MaxGroups + 1)));
    if (e == cudaSuccess) done.fetch_or(1ull << dev, std::memory_order_release);
    return e;
}

// Clusters of `parts` CTAs of the split kernel that are resident at once.
template <int BN, int AR> int resident_clusters(int dev, int parts)
{
    static std::atomic<int> n[kMaxDevices][9];
    int v = n[dev][parts].load(std::memory_order_relaxed);
    if (!v) {
        if (prepare<BN, AR, EPI_STORE, SPLIT>(dev) != cudaSuccess) return 0;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)parts;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.gridDim = dim3((unsigned)parts);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = Cfg<BN, AR, SPLIT>::kSmem + group_bytes(1);
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&v, fp8_gemm_kernel<BN, AR, EPI_STORE, SPLIT>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            v = 0;
        }
        v = v < 1 ? -1 : v;
        n[dev][parts].store(v, std::memory_order_relaxed);
    }
    return v < 0 ? 0 : v;
}

template <int BN, int AR, int E, int MODE>
cudaError_t launch(const Params &p, int dev, uint32_t grid, uint32_t parts, cudaStream_t st)
{
    cudaError_t e = prepare<BN, AR, E, MODE>(dev);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<BN, AR, MODE>::kSmem + group_bytes(p.all_groups);
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = MODE == SINGLE ? 0 : MODE == PAIR ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<BN, AR, E, MODE>, p);
}

}  // namespace
}  // namespace fp8

namespace {

// One side's fields; false when a tensor map cannot be made.
bool fill(fp8::Side &d, const Fp8Launch &L, uint32_t cols, uint32_t box_rows, bool boxes)
{
    using namespace fp8;
    const bool swiglu = L.b1 != nullptr;
    d.sa = L.sa; d.sb0 = L.sb0; d.sb1 = L.sb1;
    d.out = L.out; d.out_scales = L.out_scales; d.row_scale = L.row_scale;
    d.M = L.M; d.N = L.N;
    d.kb = (L.K + kBK - 1) / kBK;
    d.nb = (L.N + 127) / 128;
    d.n_tiles = (L.N + cols - 1) / cols;
    const size_t row = (size_t)L.N * (swiglu ? 1 : L.out_f16 ? 2 : 4);
    d.vec = row % 16 == 0 && (reinterpret_cast<uintptr_t>(L.out) & 15u) == 0;
    const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    // where no tensor map can be made of C, it is stored without
    d.boxes = boxes && !swiglu && d.vec && make_map(&d.tm_c, L.out, u8, 1, row, L.M, 128, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    const uint64_t b_rows = (uint64_t)L.groups * L.N;
    return make_map(&d.tm_a, L.a, u8, 1, L.K, L.M, kBK, box_rows, CU_TENSOR_MAP_SWIZZLE_128B) &&
           make_map(&d.tm_b0, L.b0, u8, 1, L.K, b_rows, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B) &&
           (!swiglu || make_map(&d.tm_b1, L.b1, u8, 1, L.K, b_rows, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B));
}

}  // namespace

int launch_fp8_gemm(const Fp8Launch &L, cudaStream_t st, const char **why)
{
    using namespace fp8;
    const bool swiglu = L.b1 != nullptr;
    const Fp8Launch *more = L.more && L.more->M && L.more->N ? L.more : nullptr;
    if (!L.M || !L.N || !L.groups) return more ? launch_fp8_gemm(*more, st, why) : 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev >= kMaxDevices) { *why = "device"; return 2; }
    // Row tiles at most (a group's last may be partial), of 128 rows and of a pair's 256.
    // Pairs from 1024 rows a group: 4 to 5 % faster there (4096 x 14336 x 4096: 229 against
    // 238 us, 8192^3: 514 against 540), but their 256-row tiles round groups up further (32
    // groups of 512 rows on average: 287 against 265 us; a layer with 128 rows an expert:
    // 439 against 370). M counts a layer's every assignment, negative ids among them: a rank
    // that holds few of the experts its ids name has fewer rows than this rule takes it to have.
    const uint64_t mt = L.offsets ? L.M / kBM + (L.groups < L.M ? L.groups : L.M) : (L.M + kBM - 1) / kBM;
    const uint64_t sms = (uint64_t)sm_count(dev);
    const bool few = !swiglu && !L.offsets && !more && mt * ((L.N + 255) / 256) < sms && mt * ((L.N + 127) / 128) <= sms;
    const bool pair = !few && L.M / L.groups >= 1024;
    const uint32_t cols = swiglu || few ? 128 : 256;
    Params p;
    memset(&p, 0, sizeof(p));
    // Copies of 32 rows where a group has few: 128 would bring its neighbours' rows too.
    p.box_rows = L.M / L.groups < 64 ? 32 : 128;
    if (!fill(p.side[0], L, cols, p.box_rows, pair) || (more && !fill(p.side[1], *more, cols, p.box_rows, pair))) { *why = "tensor maps"; return 2; }
    p.offsets = L.offsets;
    p.groups = L.groups;
    p.all_groups = L.groups + (more ? 1 : 0);
    p.out_f16 = L.out_f16;
    p.out_fmt = L.out_fmt;
    p.err = L.err;
    const uint32_t af = L.a_fmt == 1 ? 0u : 1u, bf = L.b_fmt == 1 ? 0u : 1u;   // FMT_E4M3 = 1, FMT_E5M2 = 2
    p.idesc = idesc_f8(pair ? 256 : 128, few ? 128 : 256, af, bf);
    if (few) {
        // Too few 128 x 256 tiles for the SMs: 128 x 128 tiles, K split over a
        // cluster as far as its CTAs all run at once and keep four blocks each.
        const uint64_t tiles = mt * p.side[0].n_tiles;
        uint32_t parts = 1;
        for (uint32_t s = 2; s <= 8; s *= 2) {
            const int fit = L.M <= 32 ? resident_clusters<128, 32>(dev, (int)s) : resident_clusters<128, 128>(dev, (int)s);
            if (tiles <= (uint64_t)fit && p.side[0].kb / s >= 4) parts = s;
        }
        const uint32_t grid = (uint32_t)(tiles * parts);
        e = L.M <= 32 ? launch<128, 32, EPI_STORE, SPLIT>(p, dev, grid, parts, st)
                      : launch<128, 128, EPI_STORE, SPLIT>(p, dev, grid, parts, st);
        if (e != cudaSuccess) { cudaGetLastError(); *why = cudaGetErrorString(e); return 2; }
        return 0;
    }
    const uint64_t rows = pair ? 256 : 128;
    uint64_t bound = (pair ? (L.offsets ? L.M / 256 + L.groups : (L.M + 255) / 256) : mt) * (uint64_t)p.side[0].n_tiles;
    if (more) bound += (more->M + rows - 1) / rows * p.side[1].n_tiles;
    if (bound >> 31) { *why = "too many tiles"; return 1; }
    const uint64_t fit = pair ? sms / 2 : sms;
    const uint32_t grid = (uint32_t)(bound < fit ? bound : fit) * (pair ? 2 : 1);
    if (pair)
        e = swiglu ? launch<256, 128, EPI_SWIGLU, PAIR>(p, dev, grid, 2, st) : launch<256, 128, EPI_STORE, PAIR>(p, dev, grid, 2, st);
    else
        e = swiglu ? launch<256, 128, EPI_SWIGLU, SINGLE>(p, dev, grid, 1, st) : launch<256, 128, EPI_STORE, SINGLE>(p, dev, grid, 1, st);
    if (e != cudaSuccess) { cudaGetLastError(); *why = cudaGetErrorString(e); return 2; }
    return 0;
}

}  // namespace mpp41
