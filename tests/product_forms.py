"""Which form a product of given sizes and strides takes, from the record of its launch on a recorder thread (no GPU)."""
import hcomm_amd as h
from hcomm_amd import HcommDataType as DT, Kernel

DIRECT_16, DIRECT_32, WAVE_32, MID_64, MID_128, TILE = range(6)

# (m, n, cols, k) by form: one, a few and more than eight ranks; rows that end inside a block and not; last stages that are full and
# not, odd numbers of stages; edges of tiles on both sides; one row and one column of results
SIZES = {
    MID_64: [(600, 700, 512, 1), (300, 1200, 1009, 3), (600, 700, 300, 10), (45, 8000, 225, 2), (640, 704, 2080, 1), (5003, 77, 520, 17)],
    MID_128: [(1500, 1600, 512, 1), (1450, 1502, 470, 2), (129, 8400, 1009, 8), (8321, 130, 225, 9), (1536, 1536, 2080, 3), (1, 17000, 260, 2)],
    TILE: [(2900, 2900, 256, 1), (2830, 2890, 225, 3), (257, 16400, 257, 2), (513, 11000, 300, 9), (1, 32600, 1009, 8), (33000, 3, 520, 1),
           (2048, 4096, 2080, 1), (300, 16300, 256, 32), (16300, 300, 767, 5)],
}


def form_of(m, n, cols, k, a_blocks=None, a_scales=None, b_blocks=None, b_scales=None):
    """a_blocks and so on: blocks (bytes of scales) that lie between two rows of each rank's matrix."""
    code, rec = h.HcommGfxRecorderThreadAlloc()
    assert code == 0
    nb, none = -(-cols // 32), [0] * k
    far = 1 << 40  # apart from one another by more than any of them is long

    def views(slot, blocks, scales):
        return h.mx_views([((slot + 2 * j) * far, (nb + blocks[j]) * 16, (slot + 2 * j + 1) * far, nb + scales[j]) for j in range(k)])
    try:
        h.check(h.HcommGfxMxProductKOnThread(rec, far, n, DT.FP32, views(2, a_blocks or none, a_scales or none),
                                             views(100, b_blocks or none, b_scales or none), k, m, n, cols))
        record, = h.launch_log(rec)
        assert record.kind == Kernel.MX_PRODUCT and record.nseg == k
        return record.rows
    finally:
        h.HcommThreadFree([rec])
