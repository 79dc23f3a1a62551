"""Every schedule of the integer product with fewer steps of K a wave than it has under way, as
many and more (whose slots are refilled), whole and ragged last steps, rows and channels that
end inside a tile, fp32 and BF16 outputs. tests/test_i8_host.py holds the list to the schedules
that the library chooses for it."""
import pytest

from test_gpu_i8 import check

pytestmark = pytest.mark.gpu

SHAPES = [
    # up to 8 rows
    (2, 17, 16), (3, 33, 128), (7, 100, 1936), (2, 17, 2048), (8, 47, 2960), (3, 17, 3200), (5, 90, 8208),
    (2, 8193, 16), (8, 8225, 128), (5, 8228, 912), (2, 8290, 1024), (7, 20001, 1008), (3, 9000, 144),
    # 16 x 16
    (9, 17, 16), (9, 17, 128), (9, 17, 1984), (9, 19, 2048), (9, 17, 3008), (10, 19, 3200),
    # 32 x 32
    (17, 4148, 16), (4243, 17, 128), (451, 273, 944), (290, 423, 1024), (426, 290, 1424), (361, 363, 1536),
    # 64 x 32
    (33, 4099, 16), (33, 4098, 128), (162, 1359, 928), (419, 577, 1024), (616, 389, 1952), (439, 580, 2048),
    # 64 x 64
    (33, 8273, 16), (17, 8753, 384), (18, 8261, 416), (20, 8499, 512), (17, 8281, 704), (18, 9404, 768),
    # 64 x 128
    (9, 16567, 144), (9, 16905, 256), (9, 17023, 400), (9, 17487, 512), (10, 16505, 656), (10, 16740, 768),
    # 128 x 128, two stages and four
    (9, 16495, 16), (9, 16401, 128), (8305, 129, 160), (8462, 149, 256), (8297, 130, 416), (8549, 136, 512),
    (66, 16774, 736), (82, 17127, 768),
    # 256 x 128
    (193, 16511, 16), (8217, 406, 128), (8347, 386, 352), (6531, 527, 384), (8489, 385, 576), (193, 16508, 768),
    # 256 x 256
    (513, 19602, 32), (647, 17021, 128), (555, 19597, 160), (646, 16531, 256), (388, 16559, 784), (388, 17073, 768),
]


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("M,O,K", SHAPES)
def test_i8_schedule(hip, rng, M, O, K, bf):
    check(hip, rng, M, O, K, hip.Y_BF16 if bf else 0)
