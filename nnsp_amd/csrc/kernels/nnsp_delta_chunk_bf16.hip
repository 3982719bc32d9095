// nnsp_delta_chunk_bf16.hip -- the gated delta rule in chunks, __bf16 tensors.
#include "nnsp_delta_chunk.h"

extern "C" int nnspk_launch_delta_chunk_bf16(const nnsp_delta_args* a, void* stream) {
    return launch_chunk<__bf16>(*a, (hipStream_t)stream);
}
