// Rows of f32, f64 or bf16 values: conversion and wide loads and stores.
#pragma once

#include "common.h"

namespace ye3t {

// The arithmetic type of a storage type: sums of bf16 rows are held in fp32.
template <typename T>
struct Wide {
  typedef float type;
};
template <>
struct Wide<double> {
  typedef double type;
};

// V values at any alignment of the value's own type.  Rows of odd widths start
// at every multiple of it; the memory pipeline takes a vector there in one
// instruction.
template <typename T, int V>
struct Chunk {
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v;
  __device__ static Chunk load(const T* p) {
    Chunk c;
    c.v = *reinterpret_cast<const vec*>(p);
    return c;
  }
  __device__ static Chunk zero() {
    Chunk c;
    c.v = vec(T(0.0f));
    return c;
  }
  __device__ void store(T* p) const { *reinterpret_cast<vec*>(p) = v; }
  // the first `n` values, the others zero
  __device__ static Chunk load(const T* p, int n) {
    if (n >= V) return load(p);
    Chunk c = zero();
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (q < n) c.v[q] = p[q];
    return c;
  }
  __device__ void store(T* p, int n) const {
    if (n >= V) {
      store(p);
      return;
    }
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (q < n) p[q] = v[q];
  }
};

// 16 bytes of one lane
template <typename T>
constexpr int kChunk = 16 / int(sizeof(T));

}  // namespace ye3t
