// Launch interface of the tcgen05 kernels with an epilogue.  They are compiled in a translation
// unit of their own (epilogue_kernels.cu); the driver (epilogue_driver.inc) fills in a launch.
#pragma once

#include "gemm_kernels.cuh"

namespace b200 {

struct EpilogueLaunch {
    int            bn;       // compiled tile width
    int            cl;       // CTAs per tile
    int            out;      // OUT_*
    bool           tr;       // transposing epilogue
    uint32_t       split;    // K partitions in a cluster (1: none)
    uint32_t       units;    // CTAs, CTA pairs or clusters
    uint32_t       smem;
    CUtensorMap    a, b, d;
    EpilogueMaps   em;
    GemmParams     gp;
    EpilogueParams ep;
};

// Shared-memory opt-in of every kernel here; loads them too.
cudaError_t set_epilogue_attributes();
cudaError_t launch_epilogue_gemm(const EpilogueLaunch& l, cudaStream_t s);
// CTA pairs that can be resident at once.
cudaError_t epilogue_pairs(int* pairs);
// Lines of `length` 16-bit elements copied to lines of `pitch` elements, zero-padded.
cudaError_t launch_pad_lines(const void* src, void* dst, uint64_t lines, uint32_t length, uint32_t pitch, const FastDiv& per_line, int sm_count, cudaStream_t s);
cudaError_t launch_ragged_maps(const CUtensorMap& a, const CUtensorMap& b, CUtensorMap* maps, const int32_t* offsets, uint32_t groups,
                               uint32_t rows, cudaStream_t s);

} // namespace b200
