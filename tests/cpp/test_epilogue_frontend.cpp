// C++ front end of the products with epilogues: each template of include/rocm_wmma_gemm/gemm.hpp runs once
// on integers small enough that every type holds every result exactly, and is compared with loops on
// the host.  Exit code 0 = all values equal.
#include <rocm_wmma_gemm/gemm.hpp>

#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace rocm_wmma_gemm;

#define CUDA_OK(x)                                                                \
    do {                                                                          \
        cudaError_t e_ = (x);                                                     \
        if (e_ != cudaSuccess) {                                                  \
            std::fprintf(stderr, "%s: %s\n", #x, cudaGetErrorString(e_));         \
            std::exit(2);                                                         \
        }                                                                         \
    } while (0)

template <class T>
struct Device {
    std::vector<T> host;
    T*             ptr = nullptr;
    explicit Device(size_t n, int seed = -1) : host(n)
    {
        for (size_t i = 0; i < n; ++i) host[i] = seed < 0 ? T(0.f) : T(float(int((i * 7 + seed) % 5) - 2));
        CUDA_OK(cudaMalloc(reinterpret_cast<void**>(&ptr), n * sizeof(T)));
        CUDA_OK(cudaMemcpy(ptr, host.data(), n * sizeof(T), cudaMemcpyHostToDevice));
    }
    ~Device() { cudaFree(ptr); }
    void back() { CUDA_OK(cudaMemcpy(host.data(), ptr, host.size() * sizeof(T), cudaMemcpyDeviceToHost)); }
    float operator[](size_t i) const { return float(host[i]); }
};

static int g_bad = 0;
static void same(const char* what, size_t i, float got, float want)
{
    if (got != want && g_bad++ < 10) std::printf("%s[%zu]: %g, not %g\n", what, i, got, want);
}
static float relu(float x) { return x > 0.f ? x : 0.f; }

template <class T, class U>
void run(cudaStream_t& s)
{
    const size_t M = 70, N = 72, K = 24, E = 3;
    const int    offs[E + 1] = {2, 30, 30, 68};
    Device<U>    A(M * K, 1), W(E * K * N, 2), G(M * N, 5);
    Device<T>    C(M * N), R(M * N, 3), Z(M * N), bias(E * N, 4), dW(E * K * N, 6);
    Device<float> bg(E * N);
    int*          off;
    CUDA_OK(cudaMalloc(reinterpret_cast<void**>(&off), sizeof(offs)));
    CUDA_OK(cudaMemcpy(off, offs, sizeof(offs), cudaMemcpyHostToDevice));
    auto dot = [&](size_t i, size_t j, size_t e) {
        float t = 0;
        for (size_t k = 0; k < K; ++k) t += A[i * K + k] * W[e * K * N + k * N + j];
        return t;
    };
    epilogue<T> e;
    e.act = activation::relu, e.bias = bias.ptr, e.residual = R.ptr, e.preact = Z.ptr;
    gemm_fused<m_layout::row_major, m_layout::row_major, m_layout::row_major>(C.ptr, A.ptr, W.ptr, M, N, K, 1, e, s);
    C.back(), Z.back();
    for (size_t i = 0; i < M * N; ++i) {
        const float z = dot(i / N, i % N, 0) + bias[i % N];
        same("fused C", i, C[i], relu(z) + R[i]);
        same("fused Z", i, Z[i], z);
    }
    epilogue<T> g;
    g.act = activation::relu, g.gradient = true, g.preact = R.ptr, g.bias_grad = bg.ptr;
    gemm_grouped<m_layout::row_major>(C.ptr, A.ptr, W.ptr, off, M, N, K, E, g, s);
    gemm_grouped_wgrad<m_layout::row_major>(dW.ptr, A.ptr, G.ptr, off, M, K, N, E, true, s);
    Device<T> before(E * K * N, 6), dz(M * N);
    C.back(), bg.back(), dW.back();
    for (size_t q = 0; q < E; ++q)
        for (size_t j = 0; j < N; ++j) {
            float sum = 0;
            for (int i = offs[q]; i < offs[q + 1]; ++i) {
                const float d = R[i * N + j] > 0.f ? dot(i, j, q) : 0.f;
                same("grouped C", i * N + j, C[i * N + j], d);
                sum += d;
            }
            same("grouped bias_grad", q * N + j, bg[q * N + j], sum);
            for (size_t k = 0; k < K; ++k) {
                float w = before[(q * K + k) * N + j];
                for (int i = offs[q]; i < offs[q + 1]; ++i) w += A[i * K + k] * G[i * N + j];
                same("wgrad", (q * K + k) * N + j, dW[(q * K + k) * N + j], w);
            }
        }
    activation_backward<m_layout::row_major>(dz.ptr, C.ptr, R.ptr, M, N, 1, activation::relu, bg.ptr, 0, nullptr, 0, s);
    dz.back(), bg.back();
    for (size_t j = 0; j < N; ++j) {
        float sum = 0;
        for (size_t i = 0; i < M; ++i) {
            const float d = R[i * N + j] > 0.f ? C[i * N + j] : 0.f;
            same("backward", i * N + j, dz[i * N + j], d);
            sum += d;
        }
        same("backward sums", j, bg[j], sum);
    }
    try {
        e.gradient = true; // with a bias: refused
        gemm_fused<m_layout::row_major, m_layout::row_major, m_layout::row_major>(C.ptr, A.ptr, W.ptr, M, N, K, 1, e, s);
        ++g_bad;
        std::printf("a bias in gradient mode was taken\n");
    } catch (const std::runtime_error&) {
    }
    cudaFree(off);
}

int main()
{
    cudaStream_t s;
    CUDA_OK(cudaStreamCreate(&s));
    run<half, half>(s);
    run<float, half>(s);
    run<__nv_bfloat16, __nv_bfloat16>(s);
    run<float, __nv_bfloat16>(s);
    CUDA_OK(cudaStreamDestroy(s));
    std::printf("%d value(s) differ\n", g_bad);
    return g_bad ? 1 : 0;
}
