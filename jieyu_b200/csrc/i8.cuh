// i8.cuh — 8-bit products with a scale for each token and each output channel (i8.cu).
#pragma once
#include "common.cuh"

namespace jyc {

struct I8Gemm {
    const int8_t* A;  // [m] rows of lda bytes
    int lda;
    const float* as;
    const int8_t* W;  // [n] rows of ldw bytes
    int ldw;
    const float* ws;
    const float* bias;  // may be null
    float* C;
    int ldc;
    int m, n, k;
};

int launch_quantize_rows(const float* x, int ldx, int rows, int k, int8_t* q, int ldq, float* scale, cudaStream_t s);
int launch_i8_gemm(const I8Gemm& g, cudaStream_t s);

}  // namespace jyc
