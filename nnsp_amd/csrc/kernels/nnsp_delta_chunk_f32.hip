// nnsp_delta_chunk_f32.hip -- the gated delta rule in chunks, float tensors.
#include "nnsp_delta_chunk.h"

extern "C" int nnspk_launch_delta_chunk_f32(const nnsp_delta_args* a, int split, void* stream) {
    return launch_chunk<float>(*a, split, (hipStream_t)stream);
}
extern "C" long long nnspk_delta_split_bytes_f32(const nnsp_delta_args* a) { return chunk_plan<float>(*a).bytes(); }
