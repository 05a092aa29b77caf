// How products of more tiles than a launch has blocks are cut, for
// tests/test_training_launches.py: host code only.
#include "../../hephaestus_amd/csrc/training_forms.hpp"

extern "C" uint64_t tiles_of_a_launch(uint64_t threads) { return hx::tiles_a_launch(threads); }
