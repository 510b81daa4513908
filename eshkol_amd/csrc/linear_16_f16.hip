/* The kernels of the linear layer and of the products by expert (linear_16.h) for f16. */
#include "linear_16.h"

int linear::run_f16(Product* q, int n, int tile, const SlopeArgs* slope, const BiasJoin* bias, char* ws, hipStream_t st) {
    return run_products<false>(q, n, tile, slope, bias, ws, st);
}
