"""The word inf is a value of the clipping's NORM_TYPE, on the command line and in files, and of no other key."""
import pytest

from yolo_amd.config import get_cfg


@pytest.mark.parametrize("word", ["inf", ".inf"])
def test_inf_is_a_norm_type(word, tmp_path):
    cfg = get_cfg()
    cfg.merge_from_list(["SOLVER.CLIP_GRADIENTS.NORM_TYPE", word])
    assert cfg.SOLVER.CLIP_GRADIENTS.NORM_TYPE == float("inf")
    cfg = get_cfg()
    cfg.SOLVER.merge_from_list(["CLIP_GRADIENTS.NORM_TYPE", word])
    assert cfg.SOLVER.CLIP_GRADIENTS.NORM_TYPE == float("inf")
    path = tmp_path / "c.yaml"
    path.write_text(f"SOLVER:\n  CLIP_GRADIENTS:\n    NORM_TYPE: {word}\n")
    cfg = get_cfg()
    cfg.merge_from_file(str(path))
    assert cfg.SOLVER.CLIP_GRADIENTS.NORM_TYPE == float("inf")


@pytest.mark.parametrize("key", ["SOLVER.BASE_LR", "SOLVER.WEIGHT_DECAY", "SOLVER.CLIP_GRADIENTS.CLIP_VALUE", "MODEL.YOLOV3.TEST_NMS_THRESH"])
@pytest.mark.parametrize("word", ["inf", ".inf", "nan"])
def test_no_other_number_is_a_word(key, word):
    cfg = get_cfg()
    node = cfg
    for k in key.split("."):
        node = node[k]
    assert isinstance(node, float)
    with pytest.raises(ValueError, match="Type mismatch"):
        cfg.merge_from_list([key, word])
