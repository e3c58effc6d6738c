// The dense layer's forward product for a few rows (axc_rows.cu).
#pragma once
#include "axc_gemm.h"

namespace axc {

struct RowsArgs {
    const void *x, *kernel;
    int rows;
    long long inputs, units, x_line, kernel_line;
    Finish fin;                                // alpha is 1
    unsigned *status;                          // cleared: nothing here waits
};

// Whether it serves the product of x [rows, inputs] and the kernel (rows: units); the scratch that it needs; the product.
bool few_rows(const Matrix &x, const Matrix &kernel);
size_t few_rows_scratch(const Matrix &x, const Matrix &kernel, const DeviceInfo &di);
int few_rows_product(const Matrix &x, const Matrix &kernel, const Finish &f, void *scratch, unsigned *status, const DeviceInfo &di, Queue &q);

}  // namespace axc
