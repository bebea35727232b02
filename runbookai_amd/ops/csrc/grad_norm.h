// What the gradient-norm kernels and their bindings share.
#pragma once

#define GRAD_CHUNK 8192   // elements a workgroup takes at a time
#define GRAD_TENSORS 128  // tensors a launch

// Passed by value as a kernel argument.  Tensor i has chunks first[i] up to
// first[i + 1], counted from the 16-byte boundary at or before its start.
struct GradTable {
    void* ptr[GRAD_TENSORS];
    long size[GRAD_TENSORS];         // elements
    int first[GRAD_TENSORS + 1];
    unsigned char kind[GRAD_TENSORS];   // 0 fp32, 1 bf16, 2 fp16
    int n;
};
