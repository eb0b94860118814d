// The LDS of a Newton-Schulz product's workgroup, byte by byte: while a wave reads the
// other groups' sums, no wave's strip may touch them, since nothing orders the two.
// Ends with 0 when every check holds.
#include "../tatara_amd/csrc/muon_tiles.hpp"

#include <cstdio>
#include <vector>

using namespace tatara;

namespace {
int failures = 0;

template <typename L>
void check(const char* name) {
    using Lds = ProductLds<L>;
    constexpr int waves = L::WR * L::WC;
    std::vector<int> reader(Lds::BYTES, -1);  // the wave that reads the byte as a sum
    for (int g = 1; g < L::KG; ++g)
        for (int w = 0; w < waves; ++w)
            for (int q = 0; q < L::TM * L::TN * 4; ++q)
                for (int lane = 0; lane < 64; ++lane)
                    for (uint32_t at = 16 * Lds::sum(g, w, q, lane), i = 0; i < 16; ++i) {
                        if (at + i >= reader.size() || reader[at + i] != -1) {
                            std::printf("%s: sum byte %u outside or held twice\n", name, at + i);
                            ++failures;
                            return;
                        }
                        reader[at + i] = w;
                    }
    using Shape = StripShape<L>;
    std::vector<int> writer(Lds::BYTES, -1);
    for (int w = 0; w < waves; ++w)
        for (int row = 0; row < 32; ++row)
            for (int i = 0; i < (Shape::PITCH - 4) * 4; ++i) {
                const uint32_t at = Lds::strip(w) + row * Shape::PITCH * 4 + i;
                const char* wrong = at >= writer.size()                       ? "outside"
                                    : writer[at] != -1                        ? "in two strips"
                                    : reader[at] != -1 && reader[at] != w     ? "read by another wave"
                                                                              : nullptr;
                if (wrong) {
                    std::printf("%s: byte %u of wave %d's strip is %s\n", name, at, w, wrong);
                    ++failures;
                    return;
                }
                writer[at] = w;
            }
}
}  // namespace

int main() {
    check<Wide>("Wide");
    check<Narrow>("Narrow");
    check<Deep>("Deep");
    check<Half>("Half");
    check<Tiny>("Tiny");
    return failures != 0;
}
