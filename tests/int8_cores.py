"""Calls of the 8-bit layer that reach every core of its sizing rule: (core, rows, inputs, channels).

Short and long sums over inputs, lengths that split unevenly over a workgroup's eight waves and that wrap the LDS
rings many times, and channels and rows that end inside a tile."""

# order of Int8Core in csrc/ops.hpp
CORES = ("decode", "rows16", "direct32x32", "direct32x64", "direct64x64", "wide128x128", "wide256x128")

CALLS = [
    ("decode", 1, 4096, 4099), ("decode", 2, 12001, 300), ("decode", 4, 8191, 129), ("decode", 8, 2047, 2051),
    ("rows16", 5, 8193, 300), ("rows16", 9, 4097, 515), ("rows16", 16, 12001, 2307),
    ("direct32x32", 20, 4097, 300), ("direct32x32", 100, 1153, 300), ("direct32x32", 96, 12001, 4099),
    ("direct32x64", 40, 4097, 5000), ("direct32x64", 129, 4097, 2307), ("direct32x64", 300, 12001, 1031),
    ("direct64x64", 48, 4096, 12288), ("direct64x64", 192, 5120, 5120), ("direct64x64", 333, 5119, 2307),
    ("direct64x64", 250, 4161, 8190),
    ("wide128x128", 1024, 4097, 4099), ("wide128x128", 1300, 12001, 2307),
    ("wide256x128", 2048, 4096, 10240), ("wide256x128", 2047, 4097, 10001), ("wide256x128", 1100, 12001, 18433),
]
