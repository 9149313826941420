// Host-callable launchers of the paged cache's kernels.
#pragma once

#include "paged_params.h"

#include <cuda_runtime.h>

namespace f2k {

// *_prepare: load the kernels on the current device, so that the first call can be a captured one.
cudaError_t kv_append_prepare(PagedType type, PagedType cache, int head_dim, bool interleaved);
// sms: of the device, here and below.
cudaError_t kv_append_launch(const AppendParams& p, PagedType type, PagedType cache, int head_dim, int sms, cudaStream_t stream);

// Query rows of a work that the token kernel's variants hold: 8, 16, 32 or 64; and the CTAs it runs with.
int         token_rows(long long rows);
int         token_ctas(int sms);
cudaError_t paged_token_prepare(PagedType type, PagedType cache, int head_dim);
// rows: of a tile, one of token_rows(); used_rows: the most that any tile of the call has.
cudaError_t paged_token_launch(const AttendParams& p, PagedType type, PagedType cache, int head_dim, int rows, int used_rows,
                               cudaStream_t stream);

// Prompts; max_new: the most new tokens of a sequence. No workspace.
cudaError_t paged_prompt_prepare(PagedType type, PagedType cache, int head_dim);
cudaError_t paged_prompt_launch(const AttendParams& p, PagedType type, PagedType cache, int head_dim, int max_new, int sms, cudaStream_t stream);

}  // namespace f2k
