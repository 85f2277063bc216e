"""Loss modules with the reference's call signatures (reference losses.py:10-106; timm LabelSmoothingCrossEntropy)."""
import torch
import torch.nn as nn

from . import ops


class LabelSmoothingCrossEntropy(nn.Module):
    """0.9*nll + 0.1*mean(-logp) (timm definition; search.py:584), one fused forward+gradient kernel."""

    def __init__(self, smoothing=0.1):
        super().__init__()
        self.smoothing = smoothing

    def forward(self, x, target):
        return ops.LabelSmoothingCE.apply(x.float(), target, float(self.smoothing))


class TopLogitsDistillation(nn.Module):
    """Distillation from a teacher of whom only the `k` largest logits of each row are kept.  `store(teacher_logits)` -> (values, classes, rest) is what a
    teacher's pass leaves (on disk, from another job, or a line above); forward(student_logits, values, classes, rest) is temperature^2 times the
    Kullback-Leibler divergence from it, averaged over the rows.  Without `rest` the stored probabilities are renormalised (ops.distill_top_logits)."""

    def __init__(self, k, temperature=1.0, reduction='mean'):
        super().__init__()
        self.k, self.temperature, self.reduction = int(k), float(temperature), reduction

    def store(self, logits):
        return ops.top_logits(logits, min(self.k, logits.shape[1]), self.temperature)

    def forward(self, logits, values, classes, rest=None):
        return ops.distill_top_logits(logits, values, classes, rest, temperature=self.temperature, reduction=self.reduction)


class DistillationLoss(nn.Module):
    """reference losses.py:10-64.  distillation_type='none' is the OFB workflow (search.py:624-631) and runs on the fused CE
    kernel; 'soft' / 'hard' follow the reference expressions on the (B, classes) logits of a model that returns
    (outputs, outputs_kd) - a handful of row-wise ATen ops on a tensor of a few hundred KB, off the search path (the OFB models
    have no distillation head, so like the reference they raise ValueError there).  'top' (not in the reference): the fused loss against the
    teacher's `top_k` largest logits (TopLogitsDistillation), on outputs_kd, or on the class logits of a model without a distillation head."""

    def __init__(self, base_criterion, teacher_model, distillation_type, alpha, tau, top_k=16):
        super().__init__()
        assert distillation_type in ['none', 'soft', 'hard', 'top']
        self.base_criterion, self.teacher_model = base_criterion, teacher_model
        self.distillation_type, self.alpha, self.tau = distillation_type, alpha, tau
        self.top = TopLogitsDistillation(top_k, tau) if distillation_type == 'top' else None

    def forward(self, inputs, outputs, labels):
        outputs_kd = None
        if not isinstance(outputs, torch.Tensor):
            outputs, outputs_kd = outputs
        base_loss = self.base_criterion(outputs, labels)
        if self.distillation_type == 'none':
            return base_loss
        if outputs_kd is None and self.distillation_type == 'top':
            outputs_kd = outputs
        if outputs_kd is None:
            raise ValueError('When knowledge distillation is enabled, the model is expected to return a Tuple[Tensor, Tensor] with the '
                             'output of the class_token and the dist_token')
        with torch.no_grad():                                            # no backprop through the teacher (losses.py:47-48)
            teacher_outputs = self.teacher_model(inputs)
            if isinstance(teacher_outputs, tuple):
                teacher_outputs = teacher_outputs[0]
        if self.distillation_type == 'top':
            distillation_loss = self.top(outputs_kd, *self.top.store(teacher_outputs.to(outputs_kd.dtype)))
        elif self.distillation_type == 'soft':                           # losses.py:50-59
            T = self.tau
            log_s = torch.log_softmax(outputs_kd.float() / T, dim=1)
            log_t = torch.log_softmax(teacher_outputs.float() / T, dim=1)
            distillation_loss = (log_t.exp() * (log_t - log_s)).sum() * (T * T) / outputs_kd.numel()
        else:                                                            # 'hard', losses.py:60-61
            logp = torch.log_softmax(outputs_kd.float(), dim=1)
            distillation_loss = -logp.gather(1, teacher_outputs.float().argmax(dim=1, keepdim=True)).mean()
        return base_loss * (1 - self.alpha) + distillation_loss * self.alpha


class OFBSearchLOSS(nn.Module):
    """reference losses.py:66-106: (base, w1*attn + w2*mlp + w3*patch + w4*embed + w5*flops)."""

    def __init__(self, base_criterion, device, attn_w=0.0001, mlp_w=0.0001, patch_w=0.0001, embedding_w=0.0001, flops_w=0.0001,
                 entropy=True, var=True, norm=True):
        super().__init__()
        self.base_criterion = base_criterion
        self.w1, self.w2, self.w3, self.w4, self.w5 = attn_w, mlp_w, patch_w, embedding_w, flops_w
        self.entropy, self.var, self.norm, self.device = entropy, var, norm, device
        self._w_vec = None

    def forward(self, inputs, outputs, labels, model, phase: str, target_flops=1.0, finish_search=False):
        if isinstance(outputs, tuple):
            raise NotImplementedError('decoder-prediction outputs are not produced by the OFB search model')
        base_loss = self.base_criterion(inputs, outputs, labels)
        if finish_search or 'arch' not in phase:
            return base_loss
        net = model.module if hasattr(model, 'module') else model
        loss_flops = net.get_flops_loss(target_flops)
        loss_attn, loss_mlp, loss_patch, loss_embedding = net.get_sparsity_loss(self.device, self.entropy, self.var, self.norm)
        go = getattr(net, '_gate_out', None)
        sp = go.get('spars') if isinstance(go, dict) else None
        if (sp is not None and sp.dim() == 1 and sp.numel() == 3 and loss_attn.data_ptr() == sp.data_ptr()
                and loss_mlp.data_ptr() == sp.data_ptr() + 4 and loss_embedding.data_ptr() == sp.data_ptr() + 8):
            # the three module terms are the slots of ONE device vector (the gate kernel's output): w1 a + w2 m + w4 e as one weighted
            # sum - 4 launches forward and 2 backward instead of 7 and ~12 (three select-backward fills and their accumulation)
            if ops._scalar_ok(loss_flops) and sp.is_cuda and sp.dtype == torch.float32 and sp.is_contiguous():
                # one launch forward, one backward (the weights are plain attributes: read at every call)
                arch = ops.ArchLoss.apply(sp, loss_flops, float(self.w1), float(self.w2), float(self.w4), float(self.w5))
            else:
                key = (float(self.w1), float(self.w2), float(self.w4), sp.device, sp.dtype)
                if self._w_vec is None or self._w_vec[0] != key:      # the weights are plain attributes: follow later edits
                    self._w_vec = (key, torch.tensor(key[:3], device=sp.device, dtype=sp.dtype))
                arch = (sp * self._w_vec[1]).sum() + self.w5 * loss_flops
        else:
            arch = self.w1 * loss_attn + self.w2 * loss_mlp + self.w4 * loss_embedding + self.w5 * loss_flops
        if self.w3 != 0:
            arch = arch + self.w3 * loss_patch
        return base_loss, arch
