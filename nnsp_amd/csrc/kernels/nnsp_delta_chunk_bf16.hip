// nnsp_delta_chunk_bf16.hip -- the gated delta rule in chunks, __bf16 tensors.
#include "nnsp_delta_chunk.h"

extern "C" int nnspk_launch_delta_chunk_bf16(const nnsp_delta_args* a, int split, void* stream) {
    return launch_chunk<__bf16>(*a, split, (hipStream_t)stream);
}
extern "C" long long nnspk_delta_split_bytes_bf16(const nnsp_delta_args* a) { return chunk_plan<__bf16>(*a).bytes(); }
