"""Values that lanes of one wave exchange through LDS need an ordering point between the stores and the other lanes' loads, and before the
next stores: the hardware keeps one wave's LDS accesses in order, the compiler need not."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tile_epilogue_orders_its_exchange():
    with open(os.path.join(ROOT, "nerffaceediting_amd", "csrc", "nfe_fp8.h")) as f:
        text = f.read()
    kernel = text[text.index("void matmul_tile_kernel("):text.index("static int tile_launch(")]
    parts = kernel[kernel.index("for (int p = 0; p < PARTS; ++p)"):]
    store, load = parts.index("*(f32x4*)(mine +"), parts.index("*(const f32x4*)(mine +")
    assert store < load
    assert len(re.findall(r"\bwave_sync\(\);", parts[:store])) == 1, "the stores of a part follow the loads of the one before"
    assert len(re.findall(r"\bwave_sync\(\);", parts[store:load])) == 1, "the loads follow the stores"
