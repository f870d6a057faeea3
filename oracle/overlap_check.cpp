// overlap_check.cpp -- test infrastructure: freetoken-rs_amd/csrc/ft_overlap.hpp
// for the host. Called by tests/test_step_memory.py through ctypes; never
// linked into the product.
#include "../freetoken-rs_amd/csrc/ft_overlap.hpp"

extern "C" int oc_overlap(uint64_t a, int64_t an, int64_t as, int64_t ab, uint64_t b, int64_t bn, int64_t bs, int64_t bb) {
    return ft::overlap({reinterpret_cast<const void*>(a), an, as, ab}, {reinterpret_cast<const void*>(b), bn, bs, bb});
}
