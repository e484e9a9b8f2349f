// Which rows of a matrix may be read as whole 16-byte words without a look at
// the matrix's ends (rownorm.cu).  Plain C++, so that a host compiler can check
// the rule over every size and alignment.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define BGNN_HD __host__ __device__ __forceinline__
#else
#define BGNN_HD inline
#endif

// A vector of eight columns starts inside its row and is read as the aligned
// words from its start, rounded down, to 8 elements and 16 bytes behind it.  So
// a row's words reach at most 15 bytes before the row and 7 elements and 16
// bytes behind it: 15 elements of two bytes, 11 of four.
constexpr uint32_t WORD_REACH = 15;

// Rows at either end of a matrix whose words may reach out of it, for rows `ld`
// elements apart (several matrices: the smallest): one from 15 columns on, up
// to 15 of a single column.
BGNN_HD uint32_t edge_rows(uint64_t ld) {
  return ld >= WORD_REACH ? 1u : (WORD_REACH + (uint32_t)ld - 1) / (uint32_t)ld;
}
BGNN_HD bool inner_row(uint64_t row, uint64_t rows, uint32_t edge) {
  return row >= edge && row + edge < rows;
}
