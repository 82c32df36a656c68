// The 8-bit linear layer through the C++ surface: the planner's answers and refusals (no GPU: nothing is launched, the addresses are never
// dereferenced), and the device-resident methods compiled against the header's tensor class.
#include "mme_hip_calculator.h"

#include <cstdio>
#include <cstring>

using MmeHip::Calculator;
using MmeHip::MMEStackException;
using MmeHip::Tensor;

static int failures = 0;
#define EXPECT(cond)                                                        \
    do                                                                      \
    {                                                                       \
        if (!(cond))                                                        \
        {                                                                   \
            std::printf("  FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            failures++;                                                     \
        }                                                                   \
    } while (0)

static void* at(uintptr_t mib) { return (void*) (mib << 20); } // stands in for a device address

// (never called: the methods' templates, instantiated)
void layer(Calculator& c, Tensor& codes, float* scales, Tensor& sum, const Tensor& x, const Tensor& gamma, const Tensor& w, const float* wScales, Tensor& out)
{
    c.rmsNormQuantizeDev(codes, scales, x, &gamma, &sum, &sum, 1e-5f);
    c.scaledGemmDev(out, codes, scales, w, wScales);
    c.quantizeRowsDev(codes, scales, x, &sum, MME_HIP_GATE_GELU_TANH);
    c.quantizeRowsDev(codes, scales, x);
}

int main()
{
    Tensor x({4096, 1, 1, 1, 1}, 2, MME_HIP_INT8, at(1)), w({4096, 14336, 1, 1, 1}, 2, MME_HIP_INT8, at(16)), y({14336, 1, 1, 1, 1}, 2, MME_HIP_BF16, at(512));
    Calculator::Form f = Calculator::planScaledGemm(y, x, w);
    EXPECT(f.largeTile == 3 && f.tileRows == 8 && f.splitK == 1);
    Tensor xl({4096, 4096, 1, 1, 1}, 2, MME_HIP_INT8, at(1)), yl({14336, 4096, 1, 1, 1}, 2, MME_HIP_BF16, at(512));
    f = Calculator::planScaledGemm(yl, xl, w);
    EXPECT(f.largeTile == 1 && f.tileRows == 256 && f.wavefronts == 8);
    Tensor xf({4096, 4096, 1, 1, 1}, 2, MME_HIP_FP8_143, at(1), 7, MME_HIP_FULL_INF_NAN), wf({4096, 14336, 1, 1, 1}, 2, MME_HIP_FP8_152, at(16), 15);
    bool refused = false;
    try
    {
        Calculator::planScaledGemm(yl, xf, wf);
    }
    catch (const MMEStackException& e)
    {
        refused = std::strstr(e.what(), "ASSUME_NONE") != nullptr;
    }
    EXPECT(refused);
    EXPECT(Calculator::planScaledGemm(yl, xf, wf, 256, MME_HIP_FP8_SPECIALS_ASSUME_NONE).largeTile == 1);
    std::printf(failures ? "%d FAILED\n" : "all ok\n", failures);
    return failures ? 1 : 0;
}
