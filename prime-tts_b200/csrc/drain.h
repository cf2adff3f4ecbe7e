// drain.h -- which fills of a ring of stages may still be in flight when two producers stop at any point.
//
// Producer A has issued its half of fills 0 .. a - 1 of the ring, B of 0 .. b - 1; fill i lies in stage
// i % stages, whose barrier completes its phase i / stages when both halves have arrived and their bytes
// have landed.  A producer issues fill i only after fill i - stages has been used, so what is in flight lies
// in the last `stages` fills of the further one.  Where only one half was issued, the barrier lacks the
// other's arrival, which whoever drains gives in its place.
#pragma once
#ifdef __CUDACC__
#define PTB_BOTH __host__ __device__ __forceinline__
#else
#define PTB_BOTH inline
#endif

namespace ptb {

struct Drain {
  int begin, end;       // fills to wait for, in this order
  int matched;          // fills from here on lack an arrival
};
PTB_BOTH Drain drain_of(int a, int b, int stages) {
  const int end = a > b ? a : b;
  return Drain{end > stages ? end - stages : 0, end, a < b ? a : b};
}
// The parity that fill i's phase is waited for with.
PTB_BOTH unsigned fill_parity(int i, int stages) { return static_cast<unsigned>(i / stages) & 1u; }

}  // namespace ptb
