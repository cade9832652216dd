"""Builds of the C ABI as they were before functions were added bind what they have."""
import older_builds

ADDED = ('z1_add_norm_forward', 'z1_add_norm_backward')
INIT = ('import faster_yoco_amd as f\nfrom faster_yoco_amd import library\n'
        "print(*(getattr(library.OPS_LIB, 'z1t_init' + s)(f._lib.LIB_PATH.encode()) for s in ('', '_block', '_matrix')))")


def test_each_part_binds_without_what_came_later(pkg, tmp_path):
    from faster_yoco_amd import _lib
    names = list(_lib.SIGNATURES)
    assert set(ADDED) < set(names) and set(_lib.MATRIX_SIGNATURES) < set(names)
    for without, codes in (((), '0 0 0'), (tuple(_lib.MATRIX_SIGNATURES), '0 0 -2'),
                           (tuple(_lib.MATRIX_SIGNATURES) + ADDED, '0 0 -2'), (('z1_norm_forward',), '0 -2 0')):
        res = older_builds.run(tmp_path, [n for n in names if n not in without], INIT)
        assert res.returncode == 0 and res.stdout.split('\n')[-2] == codes, (without, res.stdout, res.stderr)
