// Internal declarations shared by the host packer and the HIP kernels of libontovae_hip.so.
#ifndef ONTOVAE_INTERNAL_H
#define ONTOVAE_INTERNAL_H

#include "../../include/ontovae_hip.h"

#define ONTOVAE_ABI_VERSION 8

#ifdef __cplusplus
extern "C++" {
void ontovae_set_error(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
// at least ontovae_int8_linear_workspace_bytes(M, N, K) for every M <= max_M
int64_t ov_int8_linear_bytes_upto(int max_M, int N, int K);
}
#endif

#endif
