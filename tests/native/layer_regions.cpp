// layers_overlap against every pair of regions, over small strides, widths and offsets.
#include <stdio.h>

#include "kv_call.h"

int main() {
    unsigned long checked = 0, overlapping = 0;
    for (uint32_t tensors = 1; tensors <= 2; ++tensors)
        for (uint64_t layers = 1; layers <= 4; ++layers)
            for (uint64_t stride = 0; stride <= 9; ++stride)
                for (uint64_t wide = 1; wide <= 4; ++wide)
                    for (uint64_t narrow = 1; narrow <= 3; ++narrow)
                        for (uint64_t first = 0; first <= (tensors == 2 ? 12u : 0u); ++first)
                            for (uint64_t second = 0; second <= (tensors == 2 ? 12u : 0u); ++second) {
                                const uint64_t offset[2] = {first, second}, bytes[2] = {wide, narrow};
                                bool want = false;
                                for (uint64_t i = 0; i < layers * tensors; ++i)
                                    for (uint64_t j = 0; j < i; ++j) {
                                        const uint64_t a = offset[i % tensors] + i / tensors * stride,
                                                       b = offset[j % tensors] + j / tensors * stride;
                                        want |= a < b + bytes[j % tensors] && b < a + bytes[i % tensors];
                                    }
                                if (sglkv::layers_overlap(tensors, offset, bytes, layers, stride) != want) {
                                    fprintf(stderr, "%u tensors, %llu layers %llu apart, widths %llu %llu at %llu %llu: not %d\n",
                                            tensors, (unsigned long long)layers, (unsigned long long)stride,
                                            (unsigned long long)wide, (unsigned long long)narrow, (unsigned long long)first,
                                            (unsigned long long)second, !want);
                                    return 1;
                                }
                                ++checked;
                                overlapping += want;
                            }
    printf("layer regions ok: %lu, %lu overlap\n", checked, overlapping);
    return overlapping > 1000 && checked - overlapping > 1000 ? 0 : 1;
}
