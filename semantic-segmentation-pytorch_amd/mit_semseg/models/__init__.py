from .models import ModelBuilder, PolicyLoss, SegmentationModule
