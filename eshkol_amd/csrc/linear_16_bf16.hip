/* The kernels of the linear layer and of the products by expert (linear_16.h) for bf16. */
#include "linear_16.h"

int linear::run_bf16(Product* q, int n, int tile, const SlopeArgs* slope, const BiasJoin* bias, char* ws, hipStream_t st) {
    return run_products<true>(q, n, tile, slope, bias, ws, st);
}
