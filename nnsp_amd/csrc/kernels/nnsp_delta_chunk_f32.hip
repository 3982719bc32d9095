// nnsp_delta_chunk_f32.hip -- the gated delta rule in chunks, float tensors.
#include "nnsp_delta_chunk.h"

extern "C" int nnspk_launch_delta_chunk_f32(const nnsp_delta_args* a, void* stream) {
    return launch_chunk<float>(*a, (hipStream_t)stream);
}
