/* mx_index.h -- where a microscaled matrix's codes and scales stand, and how many bytes they take: plain C, used by the
 * kernels and by a host test. */
#ifndef MX_INDEX_H
#define MX_INDEX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define MX_FN __host__ __device__ __forceinline__
#else
#define MX_FN static inline
#endif

#define MX_BLOCK 32      /* columns of one scale */
#define MX_ATOM  128     /* rows, and columns, of one 512-byte group of scales */

/* Columns that a row holds: cols rounded up to whole groups of scales. */
MX_FN int64_t mx_wide(int64_t cols) { return (cols + MX_ATOM - 1) / MX_ATOM * MX_ATOM; }
MX_FN int64_t mx_pitch(int64_t cols, int bits) { return mx_wide(cols) * bits / 8; }
/* The scale byte of row r, block b (column / 32); atoms = mx_wide(cols) / 128. 128 rows x 4 blocks stand in 512 bytes as
 * the tensor core's copy into TMEM takes them: 32 lanes of 16 bytes, lane = row % 32, a word for each of the rows
 * lane, lane + 32, lane + 64, lane + 96, a byte for each block. */
MX_FN size_t mx_scale_at(int64_t r, int64_t b, int64_t atoms)
{
    return (size_t)((r / 128 * atoms + b / 4) * 512 + r % 32 * 16 + r / 32 % 4 * 4 + b % 4);
}

#endif
