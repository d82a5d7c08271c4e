// The tcgen05 kernels with an epilogue: instantiations and launches.
#include "epilogue_kernels.cuh"

#include <algorithm>

namespace b200 {

namespace {

template <int OUT, class K>
cudaError_t allow_smem(K kernel)
{
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)epilogue_smem_limit(OUT));
}

template <int BN, int CL, bool TR, bool KS>
cudaError_t set_one()
{
    cudaError_t e;
    if constexpr (KS) {
        e = allow_smem<OUT_F32>(gemm_epilogue_ksplit_kernel<BN, OUT_F32, TR>);
        if (e == cudaSuccess) e = allow_smem<OUT_F16>(gemm_epilogue_ksplit_kernel<BN, OUT_F16, TR>);
        if (e == cudaSuccess) e = allow_smem<OUT_BF16>(gemm_epilogue_ksplit_kernel<BN, OUT_BF16, TR>);
    } else {
        e = allow_smem<OUT_F32>(gemm_epilogue_kernel<BN, OUT_F32, CL, TR>);
        if (e == cudaSuccess) e = allow_smem<OUT_F16>(gemm_epilogue_kernel<BN, OUT_F16, CL, TR>);
        if (e == cudaSuccess) e = allow_smem<OUT_BF16>(gemm_epilogue_kernel<BN, OUT_BF16, CL, TR>);
    }
    return e;
}

template <int BN, int CL, bool TR, bool KS>
cudaError_t launch_one(const EpilogueLaunch& l, cudaStream_t s)
{
    cudaLaunchConfig_t  lc = {};
    const uint32_t      cluster = KS ? l.split : CL;
    lc.gridDim          = dim3(l.units * cluster);
    lc.blockDim         = dim3(EPI_THREADS);
    lc.dynamicSmemBytes = l.smem;
    lc.stream           = s;
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x                           = cluster;
    attr[0].val.clusterDim.y                           = 1;
    attr[0].val.clusterDim.z                           = 1;
    attr[1].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs                                           = attr;
    lc.numAttrs                                        = 2;
    auto go = [&](auto kernel) { return cudaLaunchKernelEx(&lc, kernel, l.a, l.b, l.d, l.em, l.gp, l.ep); };
    if constexpr (KS) {
        switch (l.out) {
            case OUT_F32: return go(gemm_epilogue_ksplit_kernel<BN, OUT_F32, TR>);
            case OUT_F16: return go(gemm_epilogue_ksplit_kernel<BN, OUT_F16, TR>);
            default: return go(gemm_epilogue_ksplit_kernel<BN, OUT_BF16, TR>);
        }
    } else {
        switch (l.out) {
            case OUT_F32: return go(gemm_epilogue_kernel<BN, OUT_F32, CL, TR>);
            case OUT_F16: return go(gemm_epilogue_kernel<BN, OUT_F16, CL, TR>);
            default: return go(gemm_epilogue_kernel<BN, OUT_BF16, CL, TR>);
        }
    }
}

} // namespace

cudaError_t set_epilogue_attributes()
{
    cudaFuncAttributes a; // (loads the kernels that need no attribute)
    cudaError_t        r = cudaFuncGetAttributes(&a, pad_lines_kernel);
    if (r == cudaSuccess) r = cudaFuncGetAttributes(&a, ragged_maps_kernel);
    if (r != cudaSuccess) return r;
    cudaError_t e = set_one<64, 1, false, false>();
    if (e == cudaSuccess) e = set_one<128, 1, false, false>();
    if (e == cudaSuccess) e = set_one<256, 1, false, false>();
    if (e == cudaSuccess) e = set_one<256, 2, false, false>();
    if (e == cudaSuccess) e = set_one<512, 2, false, false>();
    if (e == cudaSuccess) e = set_one<256, 2, true, false>();
    if (e == cudaSuccess) e = set_one<16, 1, true, false>();
    if (e == cudaSuccess) e = set_one<32, 1, true, false>();
    if (e == cudaSuccess) e = set_one<64, 1, true, false>();
    if (e == cudaSuccess) e = set_one<128, 1, false, true>();
    if (e == cudaSuccess) e = set_one<256, 1, false, true>();
    if (e == cudaSuccess) e = set_one<16, 1, true, true>();
    if (e == cudaSuccess) e = set_one<32, 1, true, true>();
    if (e == cudaSuccess) e = set_one<64, 1, true, true>();
    return e;
}

cudaError_t launch_epilogue_gemm(const EpilogueLaunch& l, cudaStream_t s)
{
    const bool ks = l.split > 1;
    if (l.tr && l.cl == 2) {
        if (l.bn == 256) return launch_one<256, 2, true, false>(l, s);
    } else if (l.tr) {
        switch (l.bn) {
            case 16: return ks ? launch_one<16, 1, true, true>(l, s) : launch_one<16, 1, true, false>(l, s);
            case 32: return ks ? launch_one<32, 1, true, true>(l, s) : launch_one<32, 1, true, false>(l, s);
            case 64: return ks ? launch_one<64, 1, true, true>(l, s) : launch_one<64, 1, true, false>(l, s);
        }
    } else if (ks) {
        switch (l.bn) {
            case 128: return launch_one<128, 1, false, true>(l, s);
            case 256: return launch_one<256, 1, false, true>(l, s);
        }
    } else if (l.cl == 2) {
        switch (l.bn) {
            case 256: return launch_one<256, 2, false, false>(l, s);
            case 512: return launch_one<512, 2, false, false>(l, s);
        }
    } else {
        switch (l.bn) {
            case 64: return launch_one<64, 1, false, false>(l, s);
            case 128: return launch_one<128, 1, false, false>(l, s);
            case 256: return launch_one<256, 1, false, false>(l, s);
        }
    }
    return cudaErrorInvalidValue; // not a compiled width
}

cudaError_t epilogue_pairs(int* pairs)
{
    cudaLaunchConfig_t q = {};
    q.gridDim            = dim3(2 * 148);
    q.blockDim           = dim3(EPI_THREADS);
    q.dynamicSmemBytes   = epilogue_smem_limit(OUT_F32);
    cudaLaunchAttribute a[1];
    a[0].id               = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = 2;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    q.attrs               = a;
    q.numAttrs            = 1;
    return cudaOccupancyMaxActiveClusters(pairs, gemm_epilogue_kernel<256, OUT_F32, 2>, &q);
}

cudaError_t launch_pad_lines(const void* src, void* dst, uint64_t lines, uint32_t length, uint32_t pitch, const FastDiv& per_line, int sm_count, cudaStream_t s)
{
    const uint64_t units  = lines * (pitch / 8);
    const unsigned blocks = (unsigned)std::min<uint64_t>((units + 255) / 256, (uint64_t)sm_count * 16);
    pad_lines_kernel<<<blocks, 256, 0, s>>>(static_cast<const uint16_t*>(src), static_cast<uint4*>(dst), units, length, per_line);
    return cudaGetLastError();
}

cudaError_t launch_ragged_maps(const CUtensorMap& a, const CUtensorMap& b, CUtensorMap* maps, const int32_t* offsets, uint32_t groups,
                               uint32_t rows, cudaStream_t s)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim            = dim3(groups);
    lc.blockDim           = dim3(32);
    lc.stream             = s;
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs                                           = attr;
    lc.numAttrs                                        = 1;
    return cudaLaunchKernelEx(&lc, ragged_maps_kernel, a, b, maps, offsets, rows);
}

} // namespace b200
