// Dense weight in 4 bits (no reference counterpart): `group` input features of an output feature
// share a binary16 scale and lowest value, W = low + scale * code, in the layout of
// et_linear_w4_f16 (et_abi.h): codes [nrow][ncol / 2] bytes, the even input feature in the low
// four bits; scales [ncol / group][nrow][2].  For the few rows of a decoding step, where a Linear
// costs what its weight costs to read.
#pragma once
#include <vector>

#include "CUDA_ptr.hpp"

class w4_mat {
  public:
    const int nrow;
    const int ncol;
    const int group;
    et::DeviceBuffer<uint8_t> codes;
    et::DeviceBuffer<half> scales;

    // codes and scales as they are: a weight quantised before (host or device memory)
    w4_mat(int _nrow, int _ncol, int _group, const uint8_t *_codes, const half *_scales)
        : nrow(_nrow), ncol(_ncol), group(checked(_nrow, _ncol, _group)), codes(_codes, (std::size_t)_nrow * _ncol / 2),
          scales(_scales, (std::size_t)(_ncol / _group) * _nrow * 2) {}
    // every weight to the nearest step of its group
    w4_mat(int _nrow, int _ncol, int _group, const et::DeviceBuffer<half> &dense)
        : nrow(_nrow), ncol(_ncol), group(checked(_nrow, _ncol, _group)), codes((std::size_t)_nrow * _ncol / 2),
          scales((std::size_t)(_ncol / _group) * _nrow * 2) {
        et::require(dense.size == (std::size_t)_nrow * _ncol, "w4_mat: the dense weight must hold nrow*ncol values");
        etChk(et_dense_to_w4_f16(reinterpret_cast<const et_f16 *>(dense.get()), codes.get(),
                                 reinterpret_cast<et_f16 *>(scales.get()), ncol, nrow, group, nullptr));
        etChk(et_device_sync());
    }
    static w4_mat from_dense(const float *W, int nrow, int ncol, int group = 64) {
        std::vector<half> h((std::size_t)nrow * ncol);
        for (std::size_t i = 0; i < h.size(); i++) h[i] = static_cast<half>(W[i]);
        return w4_mat(nrow, ncol, group, et::DeviceBuffer<half>(h));
    }
    // what the codes stand for, [nrow x ncol]
    et::DeviceBuffer<half> to_dense() const {
        et::DeviceBuffer<half> dense((std::size_t)nrow * ncol);
        etChk(et_w4_to_dense_f16(codes.get(), reinterpret_cast<const et_f16 *>(scales.get()),
                                 reinterpret_cast<et_f16 *>(dense.get()), ncol, nrow, group, nullptr));
        etChk(et_device_sync());
        return dense;
    }

  private:
    static int checked(int nrow, int ncol, int group) {
        et::require(group == 32 || group == 64 || group == 128, "w4_mat: the group must be 32, 64 or 128");
        et::require(nrow > 0 && ncol > 0 && nrow % 16 == 0 && ncol % group == 0,
                    "w4_mat: nrow must be a multiple of 16, ncol of the group");
        return group;
    }
};
