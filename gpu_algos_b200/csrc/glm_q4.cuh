// glm_q4.cuh -- models in 4 bits: layout, quantisation and prediction (glm_q4.cu).
#pragma once

#include "glm_common.cuh"

namespace glmb {

constexpr int kQ4Rows = 16;   // targets of a block of codes
constexpr int kQ4Cols = 64;   // features of a block of codes
constexpr int kQ4BlockBytes = kQ4Rows * kQ4Cols / 2;

inline int64_t q4_row_blocks(int64_t nt) { return (nt + kQ4Rows - 1) / kQ4Rows; }
// features are filled up to a multiple of 128, whole groups of either size
inline int64_t q4_col_blocks(int64_t nf) { return (nf + 2 * kQ4Cols - 1) / (2 * kQ4Cols) * 2; }
inline int64_t q4_groups(int64_t nf, int group) { return q4_col_blocks(nf) * kQ4Cols / group; }

template <typename T>
int q4_quantize(const T* M, void* codes, T* scales, int64_t nf, int64_t nt, int64_t ntasks, int group,
                cudaStream_t stream);
template <typename T>
int q4_dequantize(const void* codes, const T* scales, T* M, int64_t nf, int64_t nt, int64_t ntasks, int group,
                  cudaStream_t stream);
template <typename T>
size_t q4_predict_workspace(int64_t nf, int64_t nt, int64_t ntasks, int64_t nobs, int group);
template <typename T>
int q4_predict(const T* X, const void* codes, const T* scales, T* Yhat, int64_t nf, int64_t nt, int64_t ntasks,
               int64_t nobs, int group, void* ws, size_t ws_bytes, cudaStream_t stream);

// Many observations: glm_q4_tile.cu.  `vec`: X's rows are whole 16-byte pieces.
template <typename T>
size_t q4_tile_workspace(int64_t nf, int64_t ntasks, int64_t nobs);
template <typename T>
int q4_tile_predict(const T* X, const void* codes, const T* scales, T* Yhat, int64_t nf, int64_t nt, int64_t ntasks,
                    int64_t nobs, int group, bool vec, void* ws, size_t ws_bytes, cudaStream_t stream);

}  // namespace glmb
