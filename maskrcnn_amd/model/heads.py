"""FPN classifier head and mask head.

Replicates reference fpn_classifier_graph / build_fpn_mask_graph
(mrcnn/model.py:~905-1015):

Classifier: PyramidROIAlign(7x7) -> conv 7x7 -> 1024 (acts as fc1) + BN ->
conv 1x1 -> 1024 + BN -> class logits / softmax + per-class bbox deltas.

Mask: PyramidROIAlign(14x14) -> 4x (3x3 conv 256 + BN + ReLU) ->
deconv 2x2/2 -> 1x1 conv num_classes + sigmoid -> [B, R, C, 28, 28].

With config.CLASSIF_HEAD_NORM = "layer" the classifier's two dense layers are
LN(ReLU(x W1 + b1)) and LN(ReLU(h W2 + b2) + h), on the fused dense layer and
layer norm of maskrcnn_amd.ops; this has no counterpart in the reference.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import LayerNorm, linear_act
from .resnet import make_norm
from .roialign import PyramidROIAlign


class FPNClassifierHead(nn.Module):
    def __init__(self, config, in_channels=256):
        super().__init__()
        pool = config.POOL_SIZE
        fc = config.FPN_CLASSIF_FC_LAYERS_SIZE
        nc = config.NUM_CLASSES
        train_bn = bool(config.TRAIN_BN)
        self.roi_align = PyramidROIAlign(pool, config.IMAGE_SHAPE,
                                         mode="crop_and_resize")
        # 7x7 conv with VALID padding == fully-connected over the pooled tile.
        norm = getattr(config, "CLASSIF_HEAD_NORM", "batch")
        if norm not in ("batch", "layer"):
            raise ValueError(f"CLASSIF_HEAD_NORM {norm!r}: batch or layer")
        self.layer_norm = norm == "layer"
        self.mrcnn_class_conv1 = nn.Conv2d(in_channels, fc, pool)
        if self.layer_norm:
            self.mrcnn_class_ln1 = LayerNorm(fc)
        else:
            self.mrcnn_class_bn1 = make_norm(fc, train_bn)
        self.mrcnn_class_conv2 = nn.Conv2d(fc, fc, 1)
        if self.layer_norm:
            self.mrcnn_class_ln2 = LayerNorm(fc)
        else:
            self.mrcnn_class_bn2 = make_norm(fc, train_bn)
        self.mrcnn_class_logits = nn.Linear(fc, nc)
        self.mrcnn_bbox_fc = nn.Linear(fc, nc * 4)
        self.num_classes = nc

    def forward(self, rois, feature_maps):
        """rois [B,N,4] -> (logits [B,N,C], probs [B,N,C], bbox [B,N,C,4]).

        The 7x7-VALID conv1 and 1x1 conv2 are mathematically dense
        layers over the pooled tile — evaluated as F.linear (hipBLASLt
        GEMMs on ROCm) rather than MIOpen convs; parameters stay the
        Conv2d modules (state-dict parity with the reference naming).
        """
        B, N, _ = rois.shape
        x = self.roi_align(rois, feature_maps)           # [B*N,256,7,7]
        if self.layer_norm:
            logits, bbox = self._dense_layers(x)
            probs = F.softmax(logits, dim=-1)
            return (logits.reshape(B, N, -1), probs.reshape(B, N, -1),
                    bbox.reshape(B, N, self.num_classes, 4))
        w1 = self.mrcnn_class_conv1.weight
        x = F.linear(
            x.reshape(x.shape[0], -1),
            w1.reshape(w1.shape[0], -1).to(x.dtype),
            self.mrcnn_class_conv1.bias.to(x.dtype))     # [B*N, fc]
        x = F.relu(self._bn_vec(self.mrcnn_class_bn1, x))
        w2 = self.mrcnn_class_conv2.weight
        x = F.linear(x, w2.reshape(w2.shape[0], -1).to(x.dtype),
                     self.mrcnn_class_conv2.bias.to(x.dtype))
        x = F.relu(self._bn_vec(self.mrcnn_class_bn2, x))
        logits = self.mrcnn_class_logits(x)
        probs = F.softmax(logits, dim=-1)
        bbox = self.mrcnn_bbox_fc(x).reshape(B * N, self.num_classes, 4)
        return (logits.reshape(B, N, -1), probs.reshape(B, N, -1),
                bbox.reshape(B, N, self.num_classes, 4))

    def _dense_layers(self, x):
        """The layer-normed form: pooled tiles -> (logits, box deltas)."""
        def dense(layer, x, activation="none", residual=None):
            w = layer.weight
            return linear_act(x, w.reshape(w.shape[0], -1).to(x.dtype),
                              layer.bias.to(x.dtype), activation, residual)

        x = x.reshape(x.shape[0], -1)
        h = self.mrcnn_class_ln1(dense(self.mrcnn_class_conv1, x, "relu"))
        h = self.mrcnn_class_ln2(dense(self.mrcnn_class_conv2, h, "relu", h))
        return dense(self.mrcnn_class_logits, h), dense(self.mrcnn_bbox_fc, h)

    @staticmethod
    def _bn_vec(bn, x):
        """Apply a (Frozen)BatchNorm2d's affine/stats to a [M, C] vector
        (the 4D module applied at spatial size 1x1)."""
        return bn(x.unsqueeze(-1).unsqueeze(-1)).squeeze(-1).squeeze(-1)


class FPNMaskHead(nn.Module):
    def __init__(self, config, in_channels=256):
        super().__init__()
        nc = config.NUM_CLASSES
        train_bn = bool(config.TRAIN_BN)
        self._fused = not train_bn  # frozen BN folds into the 3x3 convs
        self.roi_align = PyramidROIAlign(config.MASK_POOL_SIZE,
                                         config.IMAGE_SHAPE,
                                         mode="crop_and_resize")
        layers = []
        for i in range(4):
            layers += [nn.Conv2d(in_channels if i == 0 else 256, 256, 3,
                                 padding=1),
                       make_norm(256, train_bn),
                       nn.ReLU(inplace=True)]
        self.convs = nn.Sequential(*layers)
        self.mrcnn_mask_deconv = nn.ConvTranspose2d(256, 256, 2, stride=2)
        self.mrcnn_mask = nn.Conv2d(256, nc, 1)

    def _conv_stack(self, x):
        """The 4x (3x3 conv + frozen-BN + ReLU) stack; each layer runs as
        one HIP MFMA kernel on GPU (14x14 maps: measured 1.19x over
        MIOpen before counting the fused BN/ReLU, profiles/r01_conv_ab.md).
        MASKRCNN_FP8_COMPUTE=1 (serving, BASELINE config #5) runs the
        folded convs at the fp8 MFMA rate with cached e4m3 weights."""
        import os
        if (self._fused and x.is_cuda and not self.training and
                os.environ.get("MASKRCNN_FP8_COMPUTE", "0") == "1"):
            return self._conv_stack_fp8(x)
        from ..ops.conv_policy import use_hip_conv3x3
        if not (self._fused and x.is_cuda and not self.training and
                use_hip_conv3x3(x.shape[0], x.shape[1], x.shape[2],
                                x.shape[3], 256)):
            return self.convs(x)
        from ..ops.conv3x3 import conv3x3_bn_relu
        for i in range(4):
            conv = self.convs[3 * i]
            bn = self.convs[3 * i + 1]
            x = conv3x3_bn_relu(x, conv.weight, conv.bias, bn.weight,
                                bn.bias, bn.running_mean, bn.running_var,
                                eps=bn.eps, relu=True)
        return x

    def _conv_stack_fp8(self, x):
        """fp8-compute stack via the MX block-scaled kernel (K=128
        mfma_scale — the 2x-rate path; the non-MX e4m3 kernel runs at
        the bf16 MFMA rate and measured 0.5x, r2_conv_ab). BN-folded
        weights are MX-quantized once and cached (static in serving;
        the cache is dropped by train() via the _fp8_cache check)."""
        from ..ops.conv3x3 import conv3x3_mx, pack_weight_mx
        if getattr(self, "_fp8_cache", None) is None:
            import torch as _t
            cache = []
            with _t.no_grad():
                for i in range(4):
                    conv = self.convs[3 * i]
                    bn = self.convs[3 * i + 1]
                    s = bn.weight * (bn.running_var + bn.eps).rsqrt()
                    w_eff = conv.weight * s.view(-1, 1, 1, 1)
                    b_eff = bn.bias + (conv.bias - bn.running_mean) * s
                    wq, ws = pack_weight_mx(w_eff)
                    cache.append((wq.to(x.device), ws.to(x.device),
                                  b_eff.float().to(x.device)))
            self._fp8_cache = cache
        for wq, ws, b_eff in self._fp8_cache:
            x = conv3x3_mx(x, wq, ws, b_eff, relu=True)
        return x

    def train(self, mode: bool = True):
        if mode:
            self._fp8_cache = None  # weights may change: drop quant cache
        return super().train(mode)

    def forward(self, rois, feature_maps):
        """rois [B,N,4] -> mask LOGITS [B,N,C,28,28].

        (The reference applies sigmoid inside the graph; we keep logits for
        an autocast-safe BCE-with-logits loss and apply sigmoid at the
        inference output — numerically identical end to end.)
        """
        B, N, _ = rois.shape
        x = self.roi_align(rois, feature_maps)           # [B*N,256,14,14]
        x = self._conv_stack(x)
        import os
        if (x.is_cuda and x.dtype == torch.bfloat16 and
                x.is_contiguous(memory_format=torch.channels_last) and
                (not self.training or
                 os.environ.get("MASKRCNN_HIP_DECONV") == "1") and
                os.environ.get("MASKRCNN_HIP_DECONV", "1") != "0"):
            # One MFMA GEMM + scatter (csrc/hip/deconv2x2.hip, N6);
            # fuses the ReLU. Eval/serving only by default: the r5
            # bench A/B measured the per-step weight re-pack + aten
            # backward mix costing ~0.7 ms/step in training (46.25 vs
            # 45.52); MASKRCNN_HIP_DECONV=1 forces it on in training,
            # =0 forces MIOpen everywhere.
            from ..ops.deconv import deconv2x2_bias_relu
            x = deconv2x2_bias_relu(x, self.mrcnn_mask_deconv.weight,
                                    self.mrcnn_mask_deconv.bias,
                                    relu=True)
        else:
            x = F.relu(self.mrcnn_mask_deconv(x))
        x = self.mrcnn_mask(x)                           # [B*N, C, 28, 28]
        return x.reshape(B, N, *x.shape[1:])
