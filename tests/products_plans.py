"""How csrc/products/plan.h cuts a product, asked on the CPU: the header is plain C++.  The lists below are calls that together take
every way through the library that the model chooses (cheap ones of some million random sizes, for each way one);
tests/test_products_plans.py holds the model to them and tests/test_gpu_products_cuts.py runs them."""

import ctypes as C
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PLAN_H = os.path.join(ROOT, "battgp_amd", "csrc", "products", "plan.h")
CUTS = ["DIRECT16", "DIRECT32", "PLAIN64", "PLAIN128", "PIPE64", "PIPE128", "PIPE256", "TWIN64"]

SOURCE = f"""
#include "{PLAN_H}"
namespace {{
int code(const Plan& p) {{ return p.cut | p.split << 4 | (p.pack ? 1 << 16 : 0); }}
}}
extern "C" int rows(int size, int64_t T, int64_t N, int64_t K, int64_t G, int trans, int ok, double bytes) {{
  return code(plan_rows(size, T, N, K, G, trans, Operands{{ok != 0, bytes}}));
}}
extern "C" int dw(int size, int64_t T, int64_t N, int64_t K, int64_t G, int ok, double bytes) {{
  return code(plan_dw(size, T, N, K, G, Operands{{ok != 0, bytes}}));
}}
extern "C" int int8(int out_bytes, int64_t M, int64_t N, int64_t K, int ok, double bytes) {{
  return code(plan_int8(out_bytes, M, N, K, Operands{{ok != 0, bytes}}));
}}
"""


class Plans:
    def __init__(self, folder):
        lib = os.path.join(folder, "plans.so")
        subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-x", "c++", "-", "-o", lib], input=SOURCE, text=True, check=True)
        self.lib = C.CDLL(lib)
        n, d, i = C.c_int64, C.c_double, C.c_int
        self.lib.rows.argtypes = [i, n, n, n, n, i, i, d]
        self.lib.dw.argtypes = [i, n, n, n, n, i, d]
        self.lib.int8.argtypes = [i, n, n, n, i, d]

    @staticmethod
    def named(code):
        """(cut, into how many parts k is split, whether operands are copied)"""
        return CUTS[code & 15], code >> 4 & 0xfff, bool(code >> 16)

    @staticmethod
    def padded(extent, size):
        return (extent * size + 127) // 128 * 128

    def rows(self, size, t, n, k, g, trans):
        """contiguous operands of torch's allocator: aligned where their rows are"""
        x_ok = k * size % 16 == 0
        w_ok = (n if trans else k) * size % 16 == 0  # (along rows no chunk may reach past a row's end either: the same)
        per, extent = (k, n) if trans else (n, k)
        nbytes = (0 if x_ok else t * self.padded(k, size)) + (0 if w_ok else g * per * self.padded(extent, size))
        return self.named(self.lib.rows(size, t, n, k, g, trans, x_ok and w_ok, nbytes))

    def dw(self, size, t, n, k, g):
        y_ok, x_ok = n * size % 16 == 0, k * size % 16 == 0
        nbytes = (0 if y_ok else t * self.padded(n, size)) + (0 if x_ok else t * self.padded(k, size))
        return self.named(self.lib.dw(size, t, n, k, g, x_ok and y_ok, nbytes))

    def int8(self, out_bytes, m, n, k):
        ok = k % 16 == 0
        return self.named(self.lib.int8(out_bytes, m, n, k, ok, 0 if ok else (m + n) * self.padded(k, 1)))


def counts(t, g):
    """rows of the groups: uneven, some without any"""
    weight = [(3, 1, 0, 5, 2)[i % 5] for i in range(g)]
    c = [t * w // sum(weight) for w in weight]
    c[0] += t - sum(c)
    return c


# of each: bytes of an element, rows, n, k, groups; the cut, into how many parts k is split, whether operands are copied, and in tiles of
# 256 into how many parts those of the last round are cut (0: there is none)
ROWS = [
    (2, 1, 8, 60, 5, "DIRECT16", 1, False, 0), (2, 6614, 19, 69, 3, "DIRECT32", 1, False, 0), (2, 1815, 2928, 64, 16, "PIPE128", 1, False, 0),
    (2, 2544, 824, 1367, 3, "PIPE128", 1, True, 0), (2, 3784, 2762, 72, 16, "PIPE256", 1, False, 1), (2, 7704, 2552, 72, 16, "PIPE256", 1, False, 2),
    (2, 10221, 1567, 72, 9, "PIPE256", 1, False, 4), (2, 8552, 1424, 141, 3, "PIPE256", 1, True, 1), (2, 17192, 2050, 70, 7, "PIPE256", 1, True, 2),
    (2, 13551, 2456, 70, 7, "PIPE256", 1, True, 4), (2, 12, 2488, 280, 16, "PIPE64", 1, False, 0), (2, 4554, 1697, 258, 3, "PIPE64", 1, True, 0),
    (2, 16, 1366, 3168, 16, "PIPE64", 2, False, 0), (2, 1039, 3329, 73, 16, "PLAIN128", 1, False, 0), (2, 6312, 71, 3307, 5, "PLAIN128", 8, False, 0),
    (2, 579, 1586, 69, 16, "PLAIN64", 1, False, 0), (2, 265, 396, 3556, 9, "PLAIN64", 8, False, 0), (2, 8, 1568, 1384, 9, "TWIN64", 1, False, 0),
    (2, 3037, 256, 970, 3, "TWIN64", 1, True, 0), (2, 1, 10, 4072, 3, "TWIN64", 16, False, 0), (4, 1, 8, 60, 5, "DIRECT16", 1, False, 0),
    (4, 6345, 17, 72, 9, "DIRECT32", 1, False, 0), (4, 7176, 976, 60, 5, "PIPE128", 1, False, 0), (4, 15918, 1736, 65, 3, "PIPE128", 1, True, 0),
    (4, 14824, 41, 72, 7, "PIPE64", 1, False, 0), (4, 4264, 3352, 67, 3, "PIPE64", 1, True, 0), (4, 1, 8, 2056, 7, "PIPE64", 16, False, 0),
    (4, 1152, 1192, 2306, 1, "PIPE64", 2, True, 0), (4, 6680, 968, 62, 16, "PLAIN128", 1, False, 0),
    (4, 3432, 1013, 2414, 5, "PLAIN128", 2, False, 0), (4, 288, 3350, 61, 9, "PLAIN64", 1, False, 0), (4, 1, 8, 2345, 7, "PLAIN64", 16, False, 0),
    (8, 1, 8, 60, 3, "DIRECT16", 1, False, 0), (8, 7592, 17, 86, 7, "DIRECT32", 1, False, 0), (8, 690, 1384, 64, 16, "PIPE64", 1, False, 0),
    (8, 5722, 1680, 61, 3, "PIPE64", 1, True, 0), (8, 1, 8, 1656, 7, "PIPE64", 16, False, 0), (8, 1, 8, 2335, 7, "PIPE64", 16, True, 0),
    (8, 7736, 915, 61, 5, "PLAIN128", 1, False, 0), (8, 4509, 728, 2853, 9, "PLAIN128", 2, False, 0), (8, 528, 2453, 73, 7, "PLAIN64", 1, False, 0),
    (8, 1, 8, 2225, 16, "PLAIN64", 16, False, 0),
]
# the weights' output axis contiguous
ROWS_TURNED = [
    (2, 1868, 2688, 64, 16, "PIPE128", 1, False, 0), (2, 872, 3944, 251, 16, "PIPE128", 1, True, 0), (2, 3132, 3352, 72, 9, "PIPE256", 1, False, 1),
    (2, 12632, 1456, 72, 16, "PIPE256", 1, False, 2), (2, 3616, 4024, 72, 9, "PIPE256", 1, False, 4), (2, 6384, 1896, 67, 3, "PIPE256", 1, True, 1),
    (2, 5432, 3648, 69, 5, "PIPE256", 1, True, 2), (2, 5216, 2520, 66, 9, "PIPE256", 1, True, 4), (2, 1, 8, 64, 5, "PIPE64", 1, False, 0),
    (2, 8, 2128, 417, 9, "PIPE64", 1, True, 0), (2, 12, 144, 2424, 16, "PIPE64", 8, False, 0), (2, 12, 136, 3206, 16, "PIPE64", 8, True, 0),
    (2, 2032, 2127, 65, 16, "PLAIN128", 1, False, 0), (2, 5813, 72, 3708, 16, "PLAIN128", 8, False, 0), (2, 1, 8, 60, 5, "PLAIN64", 1, False, 0),
    (2, 1, 9, 995, 16, "PLAIN64", 4, False, 0), (2, 1, 8, 72, 7, "TWIN64", 1, False, 0), (2, 1, 8, 324, 3, "TWIN64", 1, True, 0),
    (2, 1, 8, 1296, 3, "TWIN64", 4, False, 0), (2, 1, 8, 1287, 5, "TWIN64", 4, True, 0), (4, 1, 8, 60, 5, "DIRECT16", 1, False, 0),
    (4, 6484, 18, 80, 7, "DIRECT32", 1, False, 0), (4, 19113, 336, 64, 3, "PIPE128", 1, False, 0), (4, 19063, 366, 112, 9, "PIPE128", 1, True, 0),
    (4, 2176, 344, 60, 9, "PIPE64", 1, False, 0), (4, 232, 3304, 231, 9, "PIPE64", 1, True, 0), (4, 1, 8, 2032, 5, "PIPE64", 16, False, 0),
    (4, 11, 88, 3871, 16, "PIPE64", 16, True, 0), (4, 2629, 2738, 60, 5, "PLAIN128", 1, False, 0), (4, 14318, 200, 2779, 9, "PLAIN128", 2, False, 0),
    (4, 13992, 69, 64, 5, "PLAIN64", 1, False, 0), (4, 1, 8, 2449, 5, "PLAIN64", 16, False, 0), (8, 1, 8, 60, 7, "DIRECT16", 1, False, 0),
    (8, 6575, 23, 82, 3, "DIRECT32", 1, False, 0), (8, 261, 3952, 60, 7, "PIPE64", 1, False, 0), (8, 14155, 33, 354, 9, "PIPE64", 1, True, 0),
    (8, 1, 8, 1648, 5, "PIPE64", 16, False, 0), (8, 1, 8, 2139, 16, "PIPE64", 16, True, 0), (8, 5240, 1268, 67, 16, "PLAIN128", 1, False, 0),
    (8, 11981, 488, 3973, 3, "PLAIN128", 2, False, 0), (8, 312, 3713, 64, 7, "PLAIN64", 1, False, 0), (8, 1, 9, 2270, 9, "PLAIN64", 16, False, 0),
]
# weight gradients
DW = [
    (2, 219, 80, 3080, 16, "PIPE128", 1, False, 0), (2, 200, 3184, 516, 16, "PIPE128", 1, True, 0), (2, 18500, 3712, 80, 3, "PIPE128", 2, False, 0),
    (2, 19288, 3864, 68, 3, "PIPE128", 2, True, 0), (2, 200, 208, 3776, 16, "PIPE256", 1, False, 1), (2, 208, 656, 3192, 16, "PIPE256", 1, False, 2),
    (2, 200, 728, 2912, 16, "PIPE256", 1, False, 4), (2, 225, 464, 3700, 16, "PIPE256", 1, True, 1), (2, 200, 745, 3320, 16, "PIPE256", 1, True, 2),
    (2, 224, 673, 2852, 16, "PIPE256", 1, True, 4), (2, 18024, 1160, 2248, 3, "PIPE256", 2, False, 1),
    (2, 16864, 3208, 456, 3, "PIPE256", 4, False, 2), (2, 17192, 1088, 984, 1, "PIPE256", 16, False, 4),
    (2, 16112, 3880, 645, 3, "PIPE256", 2, True, 1), (2, 16696, 467, 2744, 3, "PIPE256", 4, True, 2), (2, 9024, 1844, 1095, 1, "PIPE256", 8, True, 4),
    (2, 200, 8, 8, 9, "PIPE64", 1, False, 0), (2, 3160, 9, 2736, 7, "PIPE64", 1, True, 0), (2, 5990, 648, 8, 3, "PIPE64", 8, False, 0),
    (2, 6592, 1600, 10, 3, "PIPE64", 4, True, 0), (2, 208, 3480, 69, 16, "PLAIN128", 1, False, 0), (2, 9910, 2130, 68, 3, "PLAIN128", 8, False, 0),
    (2, 200, 9, 8, 3, "PLAIN64", 1, False, 0), (2, 2975, 9, 9, 3, "PLAIN64", 4, False, 0), (2, 200, 8, 8, 3, "TWIN64", 1, False, 0),
    (2, 966, 8, 9, 3, "TWIN64", 1, True, 0), (2, 3901, 8, 8, 3, "TWIN64", 4, False, 0), (2, 1296, 8, 9, 1, "TWIN64", 4, True, 0),
    (4, 200, 8, 8, 5, "DIRECT16", 1, False, 0), (4, 206, 955, 19, 16, "DIRECT32", 1, False, 0), (4, 220, 3952, 80, 16, "PIPE128", 1, False, 0),
    (4, 1058, 3832, 70, 16, "PIPE128", 1, True, 0), (4, 19350, 216, 3824, 1, "PIPE128", 8, False, 0), (4, 18418, 1074, 848, 1, "PIPE128", 8, True, 0),
    (4, 233, 1824, 36, 16, "PIPE64", 1, False, 0), (4, 1517, 2736, 35, 5, "PIPE64", 1, True, 0), (4, 2064, 8, 8, 1, "PIPE64", 16, False, 0),
    (4, 5205, 8, 9, 1, "PIPE64", 16, True, 0), (4, 280, 3983, 72, 16, "PLAIN128", 1, False, 0), (4, 17350, 86, 2597, 3, "PLAIN128", 8, False, 0),
    (4, 200, 35, 1778, 16, "PLAIN64", 1, False, 0), (4, 2338, 8, 10, 1, "PLAIN64", 16, False, 0), (8, 200, 8, 8, 7, "DIRECT16", 1, False, 0),
    (8, 205, 20, 773, 16, "DIRECT32", 1, False, 0), (8, 200, 48, 1990, 16, "PIPE64", 1, False, 0), (8, 292, 2722, 173, 16, "PIPE64", 1, True, 0),
    (8, 4927, 8, 8, 3, "PIPE64", 16, False, 0), (8, 2216, 8, 9, 1, "PIPE64", 16, True, 0), (8, 208, 4008, 101, 16, "PLAIN128", 1, False, 0),
    (8, 17656, 344, 1577, 3, "PLAIN128", 4, False, 0), (8, 272, 33, 1934, 16, "PLAIN64", 1, False, 0), (8, 12676, 8, 9, 5, "PLAIN64", 16, False, 0),
    (2, 5433, 72, 1552, 16, "PIPE128", 1, False, 0), (2, 3360, 66, 2840, 9, "PIPE128", 1, True, 0), (2, 3160, 3528, 144, 16, "PIPE256", 1, False, 1),
    (2, 3264, 416, 2592, 16, "PIPE256", 1, False, 2), (2, 3152, 1416, 672, 16, "PIPE256", 1, False, 4),
    (2, 3292, 133, 3728, 16, "PIPE256", 1, True, 1), (2, 3160, 2600, 402, 16, "PIPE256", 1, True, 2), (2, 3158, 728, 1365, 16, "PIPE256", 1, True, 4),
    (4, 3008, 80, 4008, 16, "PIPE128", 1, False, 0), (4, 3680, 71, 3688, 16, "PIPE128", 1, True, 0),
]
# 8 bits: bytes written (16: 8 read as well) for a result; rows, n, k; the cut and so on
INT8 = [
    (16, 1, 1, 200, "DIRECT16", 1, False, 0), (2, 17, 4159, 216, "DIRECT32", 1, False, 0), (2, 4263, 1515, 208, "PIPE128", 1, False, 0),
    (2, 1826, 3432, 392, "PIPE128", 1, True, 0), (16, 3936, 4072, 224, "PIPE256", 1, False, 0), (2, 2458, 5108, 208, "PIPE256", 1, False, 1),
    (2, 5198, 4520, 272, "PIPE256", 1, False, 2), (2, 4930, 3767, 272, "PIPE256", 1, False, 4), (8, 3953, 4016, 246, "PIPE256", 1, True, 0),
    (2, 4264, 3007, 200, "PIPE256", 1, True, 1), (2, 4855, 4568, 285, "PIPE256", 1, True, 2), (2, 4008, 4456, 260, "PIPE256", 1, True, 4),
    (2, 5931, 66, 224, "PIPE64", 1, False, 0), (8, 644, 1527, 920, "PIPE64", 1, True, 0), (2, 5784, 518, 258, "PLAIN128", 1, False, 0),
    (2, 68, 5608, 284, "PLAIN64", 1, False, 0), (2, 4624, 37, 672, "TWIN64", 1, False, 0), (2, 270, 968, 2257, "TWIN64", 1, True, 0),
]
